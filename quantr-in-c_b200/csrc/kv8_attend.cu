// kv8_attend.cu -- attention over the 8-bit paged KV cache on the tensor cores
// (public contract: include/quantr_cuda.h).
//
// Mathematics.  The cache's codes are the tensor cores' own 8-bit integers, so
// the products are integer products (tcgen05.mma kind::i8, int32 sums, exact):
// a query row is written in fixed point as `DG` signed 8-bit digits relative to
// its largest magnitude, and a softmax weight as `DG` unsigned ones relative to
// the largest weight of its page, and each digit is a column of the product's
// second operand:
//
//   S^T (128 tokens x columns) = K (tokens x hd) . Qdigits^T
//   O^T (hd x columns)         = V^T (hd x tokens) . Wdigits^T      (per page)
//
// fp32 inputs take three digits (24 and 23 bits: no less than an fp32 product
// of the row's largest element keeps), 16-bit ones two: the step is a power of
// two near 2^-15 of the row's largest element, so that fp16 elements within
// 2^-4 and bf16 elements within 2^-7 of it are exact and smaller ones lose
// 2^-16 of it.  K and V go from memory to the tensor cores without one
// conversion.  Weights relative to their page, not to the running maximum:
// the digits then cost a page at most 2^-24 (2^-17) of its own mass, wherever
// the maximum of a long row lies, and a page has one scale, which the join
// applies once per page instead of once per token.
//
// Work is a flat list of (sequence, KV head, row tile, 128-token tile); every
// CTA takes an equal, contiguous share, so ragged batches and long sequences
// fill the GPU alike.  A row tile that several CTAs share is joined by the one
// that finishes last, in the order of the tokens (the result does not depend on
// who that is).
//
// Roles (320 threads): warps 0-3 softmax (thread = token), 4-7 join (thread =
// output element), 8 copies (TMA), 9 issues the MMAs.
#include "kv8.cuh"

#include <algorithm>
#include <cmath>
#include <cuda.h>
#include <cudaTypedefs.h>

namespace qr {
namespace {

constexpr int kThreads = 320;
constexpr int kTile = 128;     // tokens per tile
constexpr int kMeta = 16;      // ring of per-tile page scales
constexpr int kMaxStages = 6;

struct AttendParams {
    CUtensorMap kmap, vmap;
    Kv8View w;
    const void* q;
    void* out;
    float* lse;
    long long ldq, ldo;
    uint32_t type;
    int H, G, window;
    float scale2;  // scale * log2(e)
    int stages, nS, nO, tmem_cols, min_share;
    int* counters;  // one per CTA, zero between calls
    float* part;    // 2 per CTA: o [RT][128], m [RT], l [RT]
};

// ------------------------------------------------------------ tcgen05 --

__device__ __forceinline__ uint64_t desc_of(uint32_t addr, uint32_t sbo, uint32_t swizzle)
{
    uint64_t d = (uint64_t)((addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(sbo >> 4) << 32;
    d |= (uint64_t)1 << 46;  // sm_100 descriptor
    d |= (uint64_t)swizzle << 61;
    return d;
}

__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate)
{
    const uint32_t z = 0, acc = accumulate;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(z), "r"(z), "r"(z), "r"(z)
        : "memory");
}

__device__ __forceinline__ void mma_commit(uint64_t* bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(sptr(bar))
                 : "memory");
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld4(uint32_t addr, int* v)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_ld8(uint32_t addr, int* v)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(addr));
}

__device__ __forceinline__ bool elect()
{
    uint32_t pred = 0;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(pred));
    return pred != 0;
}

__device__ __forceinline__ void tma_page(const CUtensorMap* map, void* dst, int unit, uint64_t* bar)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            sptr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(0), "r"(unit), "r"(sptr(bar))
        : "memory");
}

// Every lane waits; true if all of them saw the phase.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, volatile int* abort)
{
    return __all_sync(~0u, mbar_wait_bounded(bar, parity, err, abort));
}

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Maximum over the warp, NaN if any lane has one.
__device__ __forceinline__ float warp_max_nan(float x)
{
    float y;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max_nan(float a, float b)
{
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// ---------------------------------------------------------------- the walk --

// The segments (runs of tiles of one row tile) of this CTA's share, walked by
// every warp for itself; all values are uniform over the warp.
struct Walk {
    long long pos, end, share;  // flat tiles
    long long first;            // flat index of sequence b's first tile
    int b, nrt, nt, tlo;        // row tiles, token tiles, first token tile of the sequence
    long long cnt;
    Kv8Seq s;
    // current segment
    int h, rt, t0, t1;
    long long item0;  // flat index of the row tile's first tile
};

template <int RT>
__device__ __forceinline__ long long seq_tiles(const AttendParams& p, const Kv8Seq& s, int& nrt, int& nt, int& tlo)
{
    nrt = (int)(((long long)s.n * p.G + RT - 1) / RT);
    const int have = (int)min((long long)max(s.len, 0), (long long)p.w.max_pages << p.w.lgP);
    const int low = s.len - s.n - p.window + 1;
    tlo = p.window && low > 0 ? low / kTile : 0;
    nt = max((have + kTile - 1) / kTile - tlo, 1);
    return (long long)p.w.KV * nrt * nt;
}

template <int RT>
__device__ __forceinline__ void walk_enter(const AttendParams& p, Walk& k)
{
    // pos lies in sequence b or behind it
    while (k.pos >= k.first + k.cnt) {
        k.first += k.cnt;
        ++k.b;
        k.s = kv8_seq(p.w, k.b);
        k.cnt = seq_tiles<RT>(p, k.s, k.nrt, k.nt, k.tlo);
    }
    const long long local = k.pos - k.first;
    const long long item = local / k.nt;
    const int t = (int)(local - item * k.nt);
    k.h = (int)(item / k.nrt);
    k.rt = (int)(item - (long long)k.h * k.nrt);
    k.item0 = k.pos - t;
    k.t0 = k.tlo + t;
    k.t1 = (int)min((long long)k.tlo + k.nt, k.t0 + (k.end - k.pos));
}

// The share of CTA c, and its first segment.  False: nothing to do.
template <int RT>
__device__ __forceinline__ bool walk_begin(const AttendParams& p, Walk& k)
{
    const int lane = threadIdx.x & 31;
    long long total = 0;
    int nrt, nt, tlo;
    for (int b0 = 0; b0 < p.w.B; b0 += 32) {
        long long c = 0;
        if (b0 + lane < p.w.B) c = seq_tiles<RT>(p, kv8_seq(p.w, b0 + lane), nrt, nt, tlo);
        for (int z = 16; z; z >>= 1) c += __shfl_xor_sync(~0u, c, z);
        total += c;
    }
    k.share = max((total + gridDim.x - 1) / gridDim.x, (long long)p.min_share);
    k.pos = k.share * blockIdx.x;
    k.end = min(k.pos + k.share, total);
    if (k.pos >= k.end) return false;
    // the sequence that pos lies in
    long long before = 0;
    for (int b0 = 0;; b0 += 32) {
        long long c = 0;
        if (b0 + lane < p.w.B) c = seq_tiles<RT>(p, kv8_seq(p.w, b0 + lane), nrt, nt, tlo);
        long long x = c;
        for (int d = 1; d < 32; d <<= 1) {
            const long long y = __shfl_up_sync(~0u, x, d);
            if (lane >= d) x += y;
        }
        const unsigned past = __ballot_sync(~0u, before + x > k.pos);
        if (past) {
            const int l = __ffs(past) - 1;
            k.b = b0 + l;
            k.first = before + __shfl_sync(~0u, x - c, l);
            break;
        }
        before += __shfl_sync(~0u, x, 31);
    }
    k.s = kv8_seq(p.w, k.b);
    k.cnt = seq_tiles<RT>(p, k.s, k.nrt, k.nt, k.tlo);
    walk_enter<RT>(p, k);
    return true;
}

template <int RT>
__device__ __forceinline__ bool walk_next(const AttendParams& p, Walk& k)
{
    k.pos += k.t1 - k.t0;
    if (k.pos >= k.end) return false;
    walk_enter<RT>(p, k);
    return true;
}

// ------------------------------------------------------------- shared memory --

template <int DG, int RT>
struct Shape {
    static constexpr int N = (DG * RT + 15) / 16 * 16;
    static constexpr uint32_t kPBytes = N * 128;
};

struct Bars {
    uint64_t kfull[kMaxStages], kempty[kMaxStages], vfull[kMaxStages], vempty[kMaxStages];
    uint64_t sfull[2], sempty[2], pfull[2], pempty[2], ofull[2], oempty[2], stfull[2], stempty[2];
    uint64_t mfull[kMeta], qfull, pmax[2][2], jdone, jlast;
};

struct Meta {
    float ks[4], vs[4];
    int valid;  // bit j: page j of the tile exists
    int pad[3];
};

template <int RT>
struct Small {
    Bars bars;
    Meta meta[kMeta];
    float stat_max[2][4][RT], stat_sum[2][4][RT];  // per softmax warp: its page's maximum, its own sum of weights
    float stat_vs[2][4];
    float wmax[2][4][RT];
    float qscale[2][RT];  // by the segment's parity
    int pos[2][RT];
    float join[4][5][RT];  // per join warp: the factor of what was there, then of each page
    uint32_t tmem;
    int abort;
    int last;
    int kfills[kMaxStages], vfills[kMaxStages];
};

template <int DG, int RT, int HDW>
__global__ void __launch_bounds__(kThreads, RT <= 16 ? 2 : 1) k_kv8_attend(const __grid_constant__ AttendParams p)
{
    constexpr int N = Shape<DG, RT>::N;
    constexpr uint32_t kStage = kTile * HDW, kPBytes = Shape<DG, RT>::kPBytes;
    constexpr uint32_t kSw = HDW == 128 ? 2u : 4u;  // 128- or 64-byte swizzle
    extern __shared__ uint8_t raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    const int S = p.stages;
    uint8_t* ksm = sm;
    uint8_t* vsm = sm + S * kStage;
    uint8_t* psm = vsm + S * kStage;
    uint8_t* qsm = psm + 2 * kPBytes;
    Small<RT>& z = *reinterpret_cast<Small<RT>*>(qsm + N * HDW);
    Bars& br = z.bars;
    volatile int* abort = &z.abort;
    int* err = p.w.err;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int P = p.w.P, NP = kTile >> p.w.lgP;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(&br.kfull[i], 1);
            mbar_init(&br.vfull[i], 1);
            mbar_init(&br.kempty[i], 1);
            mbar_init(&br.vempty[i], 1);
            z.kfills[i] = z.vfills[i] = 0;
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&br.sfull[i], 1);
            mbar_init(&br.sempty[i], 4);
            mbar_init(&br.pfull[i], 4);
            mbar_init(&br.pempty[i], 1);
            mbar_init(&br.ofull[i], 1);
            mbar_init(&br.oempty[i], 4);
            mbar_init(&br.stfull[i], 4);
            mbar_init(&br.stempty[i], 4);
        }
        for (int i = 0; i < kMeta; ++i) mbar_init(&br.mfull[i], 1);
        mbar_init(&br.qfull, 4);
        for (int i = 0; i < 4; ++i) mbar_init(&br.pmax[i >> 1][i & 1], P / 32);
        mbar_init(&br.jdone, 4);
        mbar_init(&br.jlast, 1);
        z.abort = 0;
        mbar_fence_init();
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sptr(&z.tmem)),
                     "r"(p.tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tm_s = z.tmem, tm_o = z.tmem + p.nS * N;
    pdl_trigger();
    pdl_wait();

    Walk k;
    const bool any = walk_begin<RT>(p, k);
    uint64_t* last_bar = nullptr;  // of the product issued last
    int last_ph = 0;
    if (any && warp == 8) {
        // ---------------------------------------------------------- copies --
        int st = 0, use = 0, mt = 0;
        bool ok = true, more = true;
        while (ok && more) {
            const int pg_end = k.t1 * NP;
            int unit = 0, nunit = 0, have = 0, nhave = 0;
            float ks = 0, vs = 0, nks = 0, nvs = 0;
            auto fetch = [&](int pg, int& u, int& hv, float& a, float& b) {
                hv = 0, u = 0, a = 0.0f, b = 0.0f;
                if (pg < pg_end && (long long)pg << p.w.lgP < k.s.len) {
                    const int x = kv8_unit(p.w, k.s, pg, k.h);
                    if (x >= 0) hv = 1, u = x, a = p.w.ks[x], b = p.w.vs[x];
                }
            };
            int pg = k.t0 * NP;
            fetch(pg + lane, nunit, nhave, nks, nvs);
            int at = 32;  // lane of the tile's first page within the fetched 32
            for (int t = k.t0; ok && t < k.t1; ++t, at += NP) {
                if (at == 32) {
                    unit = nunit, have = nhave, ks = nks, vs = nvs;
                    pg += 32;
                    fetch(pg + lane, nunit, nhave, nks, nvs);
                    at = 0;
                }
                if (use > 0 && !(ok = warp_wait(&br.kempty[st], (use - 1) & 1, err, abort))) break;
                const bool mine = lane >= at && lane < at + NP;
                const int j = lane - at;
                const unsigned valid = __ballot_sync(~0u, mine && have) >> at;
                Meta& m = z.meta[mt];
                if (mine) m.ks[j] = ks, m.vs[j] = vs;
                if (lane == at) {
                    m.valid = (int)valid;
                    z.kfills[st] += 1;
                    mbar_arrive_expect_tx(&br.kfull[st], kStage);
                }
                __syncwarp();
                if (lane == at) mbar_arrive(&br.mfull[mt]);
                if (mine) tma_page(&p.kmap, ksm + st * kStage + j * P * HDW, unit, &br.kfull[st]);
                if (use > 0 && !(ok = warp_wait(&br.vempty[st], (use - 1) & 1, err, abort))) break;
                if (lane == at) {
                    z.vfills[st] += 1;
                    mbar_arrive_expect_tx(&br.vfull[st], kStage);
                }
                __syncwarp();
                if (mine) tma_page(&p.vmap, vsm + st * kStage + j * P * HDW, unit, &br.vfull[st]);
                if (++st == S) st = 0, ++use;
                if (++mt == kMeta) mt = 0;
            }
            more = ok && walk_next<RT>(p, k);
        }
    } else if (any && warp == 9) {
        // ------------------------------------------------------------ MMAs --
        const uint32_t idS = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (8u << 24);
        const uint32_t idO = (2u << 4) | (1u << 7) | (1u << 15) | ((uint32_t)(N >> 3) << 17) | (8u << 24);
        int kst = 0, kuse = 0, vst = 0, vuse = 0, sb = 0, su = 0, pb = 0, pu = 0, ob = 0, ou = 0, seg = 0;
        const uint32_t qa = sptr(qsm), ka = sptr(ksm), va = sptr(vsm), pa = sptr(psm);
        auto issue_s = [&](bool fresh) -> bool {
            if (fresh && !warp_wait(&br.qfull, seg++ & 1, err, abort)) return false;
            if (!warp_wait(&br.kfull[kst], kuse & 1, err, abort)) return false;
            if (su > 0 && !warp_wait(&br.sempty[sb], (su - 1) & 1, err, abort)) return false;
            fence_after();
            if (elect()) {
#pragma unroll
                for (int i = 0; i < HDW / 32; ++i)
                    mma_i8(tm_s + sb * N, desc_of(ka + kst * kStage + 32 * i, 8 * HDW, kSw),
                           desc_of(qa + 32 * i, 8 * HDW, kSw), idS, i > 0);
                mma_commit(&br.sfull[sb]);
                mma_commit(&br.kempty[kst]);
            }
            __syncwarp();
            last_bar = &br.sfull[sb], last_ph = su & 1;
            if (++kst == S) kst = 0, ++kuse;
            if (++sb == p.nS) sb = 0, ++su;
            return true;
        };
        auto issue_o = [&]() -> bool {
            if (!warp_wait(&br.vfull[vst], vuse & 1, err, abort) || !warp_wait(&br.pfull[pb], pu & 1, err, abort))
                return false;
            if (ou > 0 && !warp_wait(&br.oempty[ob], (ou - 1) & 1, err, abort)) return false;
            fence_after();
            if (elect()) {
                const int per = P / 32;
#pragma unroll
                for (int i = 0; i < kTile / 32; ++i)  // 32 tokens each
                    mma_i8(tm_o + (ob * NP + i / per) * N, desc_of(va + vst * kStage + 32 * HDW * i, 8 * HDW, kSw),
                           desc_of(pa + pb * kPBytes + 32 * i, 1024, 2u), idO, i % per > 0);
                mma_commit(&br.ofull[ob]);
                mma_commit(&br.pempty[pb]);
                mma_commit(&br.vempty[vst]);
            }
            __syncwarp();
            last_bar = &br.ofull[ob], last_ph = ou & 1;
            if (++vst == S) vst = 0, ++vuse;
            if (++pb == 2) pb = 0, ++pu;
            if (++ob == p.nO) ob = 0, ++ou;
            return true;
        };
        bool ok = issue_s(true);
        while (ok) {
            for (int t = k.t0; ok && t < k.t1; ++t) {
                if (t + 1 < k.t1) ok = issue_s(false);
                ok = ok && issue_o();
            }
            if (!ok || !walk_next<RT>(p, k)) break;
            ok = issue_s(true);
        }
    } else if (any && warp < 4) {
        // --------------------------------------------------------- softmax --
        const int tid = threadIdx.x, page = tid >> p.w.lgP;
        int sb = 0, su = 0, pb = 0, pu = 0, mt = 0, mu = 0, seg = 0;
        const uint32_t tm = tm_s + ((uint32_t)warp << 21);
        constexpr float kQMax = DG == 3 ? 8323072.0f : 32512.0f;  // 127 * 256^(DG-1)
        bool ok = true, more = true;
        while (ok && more) {
            // The row tile's query rows as digits.  Its last product has read
            // the old ones (its scores have arrived).
            const int base_pos = k.s.len - k.s.n, sg = seg & 1;
            for (int r = warp; r < RT; r += 4) {
                const int f = k.rt * RT + r, qi = f / p.G, g = f - qi * p.G;
                const bool live = qi < k.s.n;
                float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                const int e = lane * 4;
                if (live && e < p.w.hd) {
                    const size_t off = (size_t)(k.s.row0 + qi) * p.ldq + (size_t)(k.h * p.G + g) * p.w.hd + e;
                    if (p.type == QUANTR_TYPE_F32)
                        load4<float>(static_cast<const float*>(p.q) + off, false, x);
                    else if (p.type == T_F16)
                        load4<__half>(static_cast<const __half*>(p.q) + off, false, x);
                    else
                        load4<__nv_bfloat16>(static_cast<const __nv_bfloat16*>(p.q) + off, false, x);
                }
                const float top = warp_max_nan(max_nan(max_nan(fabsf(x[0]), fabsf(x[1])), max_nan(fabsf(x[2]), fabsf(x[3]))));
                const bool fine = top <= 3.402823466e38f;
                // The largest power of two that keeps the row's largest element
                // in range.  Below 1e-30 every score rounds to 0 anyway.
                float inv = 0.0f, step = 0.0f;
                if (fine && top > 1e-30f) {
                    const int ex = 252 + 8 * DG - (int)(__float_as_uint(top) >> 23);
                    inv = __uint_as_float((uint32_t)ex << 23);
                    if (top * inv > kQMax) inv *= 0.5f;
                    step = 1.0f / inv;
                }
                uint32_t dig[3] = {0, 0, 0};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    int v = fine ? __float2int_rn(x[i] * inv) : 0;
#pragma unroll
                    for (int d = DG - 1; d >= 0; --d) {
                        const int lo = (int)(int8_t)v;
                        dig[d] |= (uint32_t)(lo & 255) << (8 * i);
                        v = (v - lo) >> 8;
                    }
                }
                if (e < HDW) {
#pragma unroll
                    for (int d = 0; d < DG; ++d) {
                        const int n = d * RT + r;
                        const int sw = HDW == 128 ? (n & 7) : ((n >> 1) & 3);
                        *reinterpret_cast<uint32_t*>(qsm + n * HDW + ((((e >> 4) ^ sw) << 4) | (e & 15))) = dig[d];
                    }
                }
                if (lane == 0) {
                    z.qscale[sg][r] = fine ? step * p.scale2 : __int_as_float(0x7fffffff);
                    z.pos[sg][r] = base_pos + qi;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&br.qfull);
            if (!(ok = warp_wait(&br.qfull, seg++ & 1, err, abort))) break;
            const int pos_lo = z.pos[sg][0], pos_hi = z.pos[sg][RT - 1];

            for (int t = k.t0; t < k.t1; ++t) {
                ok = warp_wait(&br.mfull[mt], mu & 1, err, abort) && warp_wait(&br.sfull[sb], su & 1, err, abort);
                if (!ok) break;
                const Meta& m = z.meta[mt];
                const float ks = m.ks[page];
                const int valid = m.valid;
                fence_after();
                float x[RT];
#pragma unroll
                for (int r0 = 0; r0 < RT; r0 += (RT < 8 ? RT : 8)) {
                    constexpr int C = RT < 8 ? RT : 8;
                    int c[DG][C];
#pragma unroll
                    for (int d = 0; d < DG; ++d) {
                        if constexpr (C == 8) tmem_ld8(tm + sb * N + d * RT + r0, c[d]);
                        else tmem_ld4(tm + sb * N + d * RT + r0, c[d]);
                    }
                    tmem_wait();
#pragma unroll
                    for (int r = 0; r < C; ++r) {
                        float v = (float)c[0][r];
#pragma unroll
                        for (int d = 1; d < DG; ++d) v = fmaf(v, 256.0f, (float)c[d][r]);
                        x[r0 + r] = v * (z.qscale[sg][r0 + r] * ks);
                    }
                }
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&br.sempty[sb]);
                const int tok = t * kTile + tid;
                if (t * kTile + kTile - 1 > pos_lo || valid != (1 << NP) - 1 ||
                    (p.window && t * kTile < pos_hi - p.window + 1)) {
                    const bool there = (valid >> page) & 1;
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const int q = z.pos[sg][r];
                        const bool seen = there && tok <= q && (!p.window || tok > q - p.window);
                        x[r] = seen ? x[r] : -INFINITY;
                    }
                }
                float mx[RT];
#pragma unroll
                for (int r = 0; r < RT; ++r) mx[r] = warp_max_nan(x[r]);
                if (P > 32) {  // the page spans several warps
                    const int w0 = P == 64 ? warp & 2 : 0, wn = P / 32;
                    if (lane == 0) {
#pragma unroll
                        for (int r = 0; r < RT; ++r) z.wmax[pb][warp][r] = mx[r];
                        mbar_arrive(&br.pmax[pb][w0 >> 1]);
                    }
                    if (!(ok = warp_wait(&br.pmax[pb][w0 >> 1], pu & 1, err, abort))) break;
                    for (int w = w0; w < w0 + wn; ++w) {
#pragma unroll
                        for (int r = 0; r < RT; ++r) mx[r] = max_nan(mx[r], z.wmax[pb][w][r]);
                    }
                }
                if (pu > 0) {
                    ok = warp_wait(&br.pempty[pb], (pu - 1) & 1, err, abort) &&
                         warp_wait(&br.stempty[pb], (pu - 1) & 1, err, abort);
                    if (!ok) break;
                }
                uint8_t* pt = psm + pb * kPBytes + (tid & 15);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    // Weight of the token relative to its page's largest.  1 + w
                    // holds w to 23 bits in its low bits, 128 + w to 16.  With
                    // two digits the largest weight is 65535/65536.
                    const float ref = mx[r] == -INFINITY ? 0.0f : mx[r];
                    const float w = ex2(DG == 3 ? x[r] - ref : x[r] - ref - 2.2013990e-5f);
                    const uint32_t u = __float_as_uint(1.0f + w);
                    const uint32_t d = DG == 3 ? u : __float_as_uint(128.0f + w);
                    const int n0 = r, sw = (tid >> 4) ^ (r & 7);
                    if constexpr (DG == 3) {
                        pt[(n0)*128 + sw * 16] = (uint8_t)((d >> 16) - 0x80);
                        pt[(n0 + RT) * 128 + ((tid >> 4) ^ ((n0 + RT) & 7)) * 16] = (uint8_t)(d >> 8);
                        pt[(n0 + 2 * RT) * 128 + ((tid >> 4) ^ ((n0 + 2 * RT) & 7)) * 16] = (uint8_t)d;
                    } else {
                        pt[(n0)*128 + sw * 16] = (uint8_t)(d >> 8);
                        pt[(n0 + RT) * 128 + ((tid >> 4) ^ ((n0 + RT) & 7)) * 16] = (uint8_t)d;
                    }
                    const uint32_t sum = __reduce_add_sync(~0u, u - 0x3f800000u);
                    if (lane == 0) {
                        z.stat_sum[pb][warp][r] = (float)sum * (1.0f / 8388608.0f);
                        z.stat_max[pb][warp][r] = mx[r];
                    }
                }
                if (tid < NP) z.stat_vs[pb][tid] = m.vs[tid];
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&br.pfull[pb]);
                    mbar_arrive(&br.stfull[pb]);
                }
                if (++sb == p.nS) sb = 0, ++su;
                if (++pb == 2) pb = 0, ++pu;
                if (++mt == kMeta) mt = 0, ++mu;
            }
            more = ok && walk_next<RT>(p, k);
        }
    } else if (any && warp < 8) {
        // ------------------------------------------------------------ join --
        const int tid = threadIdx.x - 128, w4 = warp - 4;
        const uint32_t tm = tm_o + ((uint32_t)w4 << 21);
        int sb = 0, su = 0, ob = 0, ou = 0, parts = 0;
        bool ok = true, more = true;
        constexpr float kUnit = DG == 3 ? 1.0f / 8388608.0f : 1.0f / 65536.0f;
        while (ok && more) {
            float o[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) o[r] = 0.0f;
            float m_run = -INFINITY, l_run = 0.0f;  // lane r: of row r
            for (int t = k.t0; t < k.t1; ++t) {
                if (!(ok = warp_wait(&br.stfull[sb], su & 1, err, abort))) break;
                if (lane < RT) {
                    float mp[4], mn = m_run;
                    const int per = P / 32;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        mp[j] = j < NP ? z.stat_max[sb][j * per][lane] : -INFINITY;
                        mn = max_nan(mn, mp[j]);
                    }
                    const float ref = mn == -INFINITY ? 0.0f : mn;
                    const float a = ex2(m_run - ref);
                    l_run *= a;
                    z.join[w4][0][lane] = a;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (j < NP) {
                            const float f = ex2(mp[j] - ref);
                            float sum = 0.0f;
                            for (int w = j * per; w < (j + 1) * per; ++w) sum += z.stat_sum[sb][w][lane];
                            l_run = fmaf(sum, f, l_run);
                            // A page that is masked altogether counts nothing, whatever its scale.
                            z.join[w4][1 + j][lane] = mp[j] == -INFINITY ? 0.0f : f * kUnit * z.stat_vs[sb][j];
                        }
                    m_run = mn;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&br.stempty[sb]);
                if (!(ok = warp_wait(&br.ofull[ob], ou & 1, err, abort))) break;
                fence_after();
#pragma unroll
                for (int r = 0; r < RT; ++r) o[r] *= z.join[w4][0][r];
                for (int j = 0; j < NP; ++j) {
#pragma unroll
                    for (int r0 = 0; r0 < RT; r0 += (RT < 8 ? RT : 8)) {
                        constexpr int C = RT < 8 ? RT : 8;
                        int c[DG][C];
#pragma unroll
                        for (int d = 0; d < DG; ++d) {
                            if constexpr (C == 8) tmem_ld8(tm + (ob * NP + j) * N + d * RT + r0, c[d]);
                            else tmem_ld4(tm + (ob * NP + j) * N + d * RT + r0, c[d]);
                        }
                        tmem_wait();
#pragma unroll
                        for (int r = 0; r < C; ++r) {
                            float v = (float)c[0][r];
#pragma unroll
                            for (int d = 1; d < DG; ++d) v = fmaf(v, 256.0f, (float)c[d][r]);
                            o[r0 + r] = fmaf(v, z.join[w4][1 + j][r0 + r], o[r0 + r]);
                        }
                    }
                }
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&br.oempty[ob]);
                if (++sb == 2) sb = 0, ++su;
                if (++ob == p.nO) ob = 0, ++ou;
            }
            if (!ok) break;
            // Whole row tile: write it.  Part of one: leave it in the
            // workspace, and join all parts if this is the last to come.
            const long long item1 = k.item0 + k.nt;
            const int c0 = (int)(k.item0 / k.share), c1 = (int)((item1 - 1) / k.share);
            float l[RT], mrow[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                l[r] = __shfl_sync(~0u, l_run, r);
                mrow[r] = __shfl_sync(~0u, m_run, r);
            }
            bool write = true;
            if (c0 != c1) {
                constexpr int kPart = RT * 130;
                float* mine = p.part + (size_t)(2 * blockIdx.x + ((int)blockIdx.x == c0 ? 1 : 0)) * kPart;
#pragma unroll
                for (int r = 0; r < RT; ++r) mine[r * 128 + tid] = o[r];
                if (w4 == 0 && lane < RT) mine[RT * 128 + lane] = m_run, mine[RT * 129 + lane] = l_run;
                __threadfence();
                __syncwarp();
                if (lane == 0) mbar_arrive(&br.jdone);
                if (tid == 0 && mbar_wait_bounded(&br.jdone, parts & 1, err, abort)) {
                    const int n = atomicAdd(p.counters + c0, 1);
                    z.last = n == c1 - c0;
                    if (z.last) p.counters[c0] = 0;
                    __threadfence();
                    mbar_arrive(&br.jlast);
                }
                __syncwarp();
                if (!(ok = warp_wait(&br.jlast, parts++ & 1, err, abort))) break;
                write = z.last;
                if (write) {
                    float mall[RT];
#pragma unroll
                    for (int r = 0; r < RT; ++r) mall[r] = -INFINITY, l[r] = 0.0f, o[r] = 0.0f;
                    for (int c = c0; c <= c1; ++c) {
                        const float* part = p.part + (size_t)(2 * c + (c == c0 ? 1 : 0)) * kPart;
#pragma unroll
                        for (int r = 0; r < RT; ++r) {
                            const float mp = __ldcg(part + RT * 128 + r), lp = __ldcg(part + RT * 129 + r);
                            const float mn = max_nan(mall[r], mp), ref = mn == -INFINITY ? 0.0f : mn;
                            const float a = ex2(mall[r] - ref), f = ex2(mp - ref);
                            l[r] = fmaf(lp, f, l[r] * a);
                            o[r] = fmaf(__ldcg(part + r * 128 + tid), f, o[r] * a);
                            mall[r] = mn;
                        }
                    }
#pragma unroll
                    for (int r = 0; r < RT; ++r) mrow[r] = mall[r];
                }
            }
            if (write) {
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const int f = k.rt * RT + r, qi = f / p.G, g = f - qi * p.G;
                    if (qi >= k.s.n) continue;
                    const size_t row = (size_t)k.s.row0 + qi;
                    const int hq = k.h * p.G + g;
                    const bool none = mrow[r] == -INFINITY;
                    if (tid < p.w.hd) {
                        const float v = none ? 0.0f : o[r] / l[r];
                        const size_t off = row * p.ldo + (size_t)hq * p.w.hd + tid;
                        if (p.type == QUANTR_TYPE_F32) static_cast<float*>(p.out)[off] = v;
                        else if (p.type == T_F16) static_cast<__half*>(p.out)[off] = __float2half_rn(v);
                        else static_cast<__nv_bfloat16*>(p.out)[off] = __float2bfloat16_rn(v);
                    }
                    if (p.lse && tid == 0)
                        p.lse[row * p.H + hq] =
                            none ? -INFINITY
                                 : (mrow[r] + log2f(l[r]) + (DG == 3 ? 0.0f : 2.2013990e-5f)) * 0.693147180559945f;
                }
            }
            more = walk_next<RT>(p, k);
        }
    }

    __syncthreads();
    if (z.abort && threadIdx.x == 0) {
        // Some role gave up: let the copies in flight land (bounded) before the
        // shared memory goes.
        for (int i = 0; i < S; ++i) {
            if (z.kfills[i] > 0) mbar_wait_bounded(&br.kfull[i], (z.kfills[i] - 1) & 1, nullptr);
            if (z.vfills[i] > 0) mbar_wait_bounded(&br.vfull[i], (z.vfills[i] - 1) & 1, nullptr);
        }
    }
    if (warp == 9) {
        // The products issued last are complete before their TMEM goes.
        if (last_bar) mbar_wait_bounded(last_bar, (uint32_t)last_ph, nullptr);
        __syncwarp();
    }
    fence_before();
    __syncthreads();
    if (warp == 9) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(z.tmem), "r"(p.tmem_cols) : "memory");
    }
}

// --------------------------------------------------------------- host side --

int pick_rt(const quantr_kv8_batch* b, int G)
{
    const long long rows = (long long)b->max_rows * G;
    return rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
}

struct Plan {
    int stages, nS, nO, cols, occ, grid;
    size_t smem;
};

template <int DG, int RT, int HDW>
Plan make_plan(int lgP)
{
    constexpr int N = Shape<DG, RT>::N;
    const int NP = kTile >> lgP;
    Plan r{};
    // Two buffers of scores and of outputs where 256 TMEM columns hold them
    // (two CTAs per SM), else fewer outputs, else one CTA per SM.
    const int tries[4][3] = {{2, 2, 256}, {2, 1, 256}, {2, 1, 512}, {1, 1, 512}};
    for (auto& t : tries) {
        r.nS = t[0], r.nO = t[1];
        const int need = N * (t[0] + t[1] * NP);
        if (need > t[2]) continue;
        for (r.cols = 32; r.cols < need;) r.cols *= 2;
        r.occ = r.cols <= 256 ? 2 : 1;
        break;
    }
    const size_t fixed = 1024 + 2 * Shape<DG, RT>::kPBytes + N * HDW + sizeof(Small<RT>);
    const size_t room = (r.occ == 2 ? 113 : 226) * 1024;
    r.stages = (int)std::min<size_t>(kMaxStages, (room - fixed) / (2 * kTile * HDW));
    r.smem = fixed + (size_t)r.stages * 2 * kTile * HDW;
    r.grid = r.occ * device_sm_count();
    return r;
}

bool encode_map(CUtensorMap* map, const void* base, const quantr_kv8_pool* p, int hdw)
{
    static PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
        PFN_cuTensorMapEncodeTiled_v12000 f = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", (void**)&f, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return f;
    }();
    if (!encode) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)p->head_dim, (cuuint64_t)p->page_tokens,
                                (cuuint64_t)p->n_pages * p->n_layers * p->n_kv_heads};
    const cuuint64_t strides[2] = {(cuuint64_t)p->head_dim, (cuuint64_t)p->head_dim * p->page_tokens};
    const cuuint32_t box[3] = {(cuuint32_t)hdw, (cuuint32_t)p->page_tokens, 1}, estr[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, hdw == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DG, int RT, int HDW>
cudaError_t run(AttendParams& p, const quantr_kv8_pool* pool, void* ws, const LaunchCfg& c)
{
    const Plan r = make_plan<DG, RT, HDW>(p.w.lgP);
    static int configured = -1;
    cudaError_t e = ensure_smem_attr(k_kv8_attend<DG, RT, HDW>, 227 * 1024, configured);
    if (e != cudaSuccess) return e;
    if (!encode_map(&p.kmap, pool->k, pool, HDW) || !encode_map(&p.vmap, pool->v, pool, HDW))
        return cudaErrorNotSupported;
    p.stages = r.stages, p.nS = r.nS, p.nO = r.nO, p.tmem_cols = r.cols, p.min_share = 2;
    p.counters = static_cast<int*>(ws);
    p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + 4096);
    return launch_ex(k_kv8_attend<DG, RT, HDW>, dim3(r.grid), kThreads, r.smem, c, p);
}

template <int DG, int HDW>
cudaError_t run_rt(int rt, AttendParams& p, const quantr_kv8_pool* pool, void* ws, const LaunchCfg& c)
{
    switch (rt) {
    case 4: return run<DG, 4, HDW>(p, pool, ws, c);
    case 8: return run<DG, 8, HDW>(p, pool, ws, c);
    case 16: return run<DG, 16, HDW>(p, pool, ws, c);
    default: return run<DG, 32, HDW>(p, pool, ws, c);
    }
}

} // namespace
} // namespace qr

extern "C" {

using namespace qr;

size_t quantr_kv8_attend_workspace_bytes(const quantr_kv8_pool* pool, const quantr_kv8_batch* batch, int n_heads,
                                         int max_len)
{
    (void)max_len;
    if (!pool || !batch || pool->n_kv_heads <= 0 || n_heads <= 0) return 0;
    // A counter per CTA, then two parts per CTA (at most 2 CTAs per SM).
    return 4096 + (size_t)2 * 2 * device_sm_count() * pick_rt(batch, n_heads / pool->n_kv_heads) * 130 * 4;
}

int quantr_kv8_attend_dev(void* out, long long ldo, const void* q, long long ldq, uint32_t type, int n_heads,
                          const quantr_kv8_pool* pool, const quantr_kv8_tables* tables,
                          const quantr_kv8_batch* batch, int layer, float scale, int window, int max_len, float* lse,
                          void* workspace, size_t workspace_bytes, void* stream)
{
    int rc = kv8_check_call(pool, tables, batch, layer, type);
    if (rc) return rc;
    if (n_heads <= 0 || n_heads % pool->n_kv_heads || window < 0 || max_len < 0 || !std::isfinite(scale))
        return QUANTR_ERR_BAD_ARG;
    if (batch->B == 0 || batch->max_rows == 0) return QUANTR_OK;
    const long long need = (long long)n_heads * pool->head_dim;
    if ((rc = kv8_check_rows(out, ldo, need)) || (rc = kv8_check_rows(q, ldq, need))) return rc;
    if (!workspace || ((uintptr_t)workspace & 255) ||
        workspace_bytes < quantr_kv8_attend_workspace_bytes(pool, batch, n_heads, max_len))
        return QUANTR_ERR_WORKSPACE;
    AttendParams p{};
    p.w = kv8_view(pool, tables, batch, layer);
    p.q = q, p.out = out, p.lse = lse, p.ldq = ldq, p.ldo = ldo, p.type = type;
    p.H = n_heads, p.G = n_heads / pool->n_kv_heads, p.window = window;
    p.scale2 = (float)((double)scale * 1.4426950408889634);
    LaunchCfg c;
    c.stream = (cudaStream_t)stream;
    const int rt = pick_rt(batch, p.G);
    cudaError_t e;
    if (type == QUANTR_TYPE_F32)
        e = pool->head_dim <= 64 ? run_rt<3, 64>(rt, p, pool, workspace, c) : run_rt<3, 128>(rt, p, pool, workspace, c);
    else
        e = pool->head_dim <= 64 ? run_rt<2, 64>(rt, p, pool, workspace, c) : run_rt<2, 128>(rt, p, pool, workspace, c);
    return kv8_done(e);
}

} // extern "C"
