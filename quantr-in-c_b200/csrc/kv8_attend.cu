// kv8_attend.cu -- attention over the 8-bit paged KV cache on the tensor cores
// (public contract: include/quantr_cuda.h).
//
// Mathematics.  The cache's codes are the tensor cores' own 8-bit integers, so
// the products are integer products (tcgen05.mma kind::i8, int32 sums, exact):
// a query row is written in fixed point as three signed 8-bit digits relative to
// its largest magnitude, and a softmax weight as three unsigned ones relative to
// the largest weight of its page, and each digit is a column of the product's
// second operand:
//
//   S^T (128 tokens x columns) = K (tokens x hd) . Qdigits^T
//   O^T (hd x columns)         = V^T (hd x tokens) . Wdigits^T      (per page)
//
// These are the only roundings that the integers add, the same for all types of
// queries: an element is kept to 2^-23 of its row's largest (fp16 elements within
// 2^-11 and bf16 ones within 2^-14 of it exactly), a weight to 2^-24 of its page's
// largest, so a page's output is off by up to page_tokens * 2^-24 of that weight
// times its largest value, and the weights' sum adds the same numbers.
// Two digits for 16-bit types would save 1 to 12 % (64-token chunks 53.1 -> 47.0
// us, 512 tokens 271 -> 251, long contexts 88.4 -> 87.0), but beside a token that
// has most of the weight they lose all others below 2^-17 of it, and queries with
// one large element lose their small ones.  K and V go from memory to the tensor
// cores without one conversion.  Weights are relative to their page, not to the
// running maximum: what the digits cost a page does not depend on where the
// maximum of a long row lies, and a page has one scale, which the join applies
// once per page instead of once per token.
//
// Work is shared out in (sequence, KV head, row tile of up to 16 rows) x
// 128-token tiles; see walk_begin.  A row tile that several CTAs share is joined
// by the one that finishes last, in the order of the tokens (the result does not
// depend on who that is).
//
// Roles (320 threads, two CTAs per SM): warps 0-3 softmax (thread = token), 4-7
// join (thread = output element), 8 copies (TMA, up to 6 stages ahead), 9 issues
// the MMAs.  S has two TMEM buffers (one under 16 rows and pages of 32 tokens), so
// a tile's scores are computed while the tile before is weighted, and its outputs
// while the next is scored.
//
// What bounds it, and what it measured (B200, 6.54 TB/s copy; launches back to
// back in a graph, inputs in rotation):
//   8 sequences of 200 to 262 thousand tokens, 32/4 heads of 128, bf16: 1.87 GB
//     in 286 us, 6.5 TB/s: memory.  4 of 100 to 131 thousand (459 MB): 88.4 us,
//     5.2 TB/s; the 18 us above the copy rate are launch, start (length, page
//     entry and keys are loads that wait for one another) and the join of the
//     18 to 20 CTAs that share a row tile.
//   64 sequences of 640 to 1152 tokens, fp32 (61 MB): 20.0 us, 3.1 TB/s; the start
//     and the longest CTA's tiles, one after the other.
//   1 sequence of 513 tokens: 8.6 us; latency, of one tile and the join of five.
//   6 prompt chunks of 64 tokens (2.2 GFLOP): 52.9 us.  512 tokens after 3584 (32
//     GFLOP): 270 us.  A tile takes some 4000 cycles (clock readings, with two
//     digits), nearly all in the softmax warps, of which two CTAs per SM keep two
//     in flight: a thread has one token and goes through 16 rows, each with two
//     warp-wide reductions and stores of single bytes.  No pipe is full (issue
//     slots 55 to 58 %, tensor 5 to 9 %, ex2 and conversions 6 to 7 %); the kernels
//     of 16 rows spill 36 to 116 bytes at their 96 registers.
// Tried and not kept, each beside what it was at that step, in us: one reference
// weight per warp's 32 tokens instead of per page (no exchange between warps, but
// four outputs per tile to join: long contexts 94 -> 103); scoring a tile ahead
// of the weights, which then wait for the next tile's keys (94 -> 108); row tiles
// of 32, whose registers leave one CTA per SM (chunks of 64 fp32 rows 67 -> 83).
#include "kv8.cuh"
#include "kv8_join.cuh"

#include <algorithm>
#include <cmath>
#include <cuda.h>
#include <cudaTypedefs.h>

namespace qr {
namespace {

constexpr int kThreads = 320;
constexpr int kTile = 128;     // tokens per tile
constexpr int kMeta = 16;      // rings of the segments, and of the tiles' page scales
constexpr int kMaxStages = 6;
// Tiles that sharing out by row tiles may cost the longest CTA.  With 0, 64 sequences
// of 640 to 1152 tokens take 26.5 us instead of 20.0; with 2, 16 of 1000 to 2000
// with 16 KV heads 27.2 instead of 24.5; with 12, 20 of 2000 to 8000 36.7 instead
// of 32.8; always by row tiles, 8 of 500 to 100,000 75.5 instead of 54.6.
constexpr int kSlack = 5;

struct AttendParams {
    CUtensorMap kmap, vmap;
    Kv8View w;
    const void* q;
    void* out;
    float* lse;
    long long ldq, ldo;
    int H, G, window;
    unsigned inv_g;  // ceil(2^32 / G): f / G = umulhi(f, inv_g) for f * G < 2^32 (G = 1 apart)
    float scale2;  // scale * log2(e)
    int vec;       // query rows allow aligned loads of four
    int stages, nS, nO, tmem_cols;
    int* counters;  // see kv8_join.cuh; zero between calls
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

// One segment: a run of 128-token tiles of one row tile.  c0, c1: the first and
// last CTA that have a part of the row tile.
struct Seg {
    int h, rt, row0, n, len;  // KV head, row tile; the sequence's first row, rows, length
    int t0, t1, c0, c1;       // t1 = t0: no more segments
};

// The copying warp walks this CTA's share; all values are uniform over it.
struct Walk {
    int pos, end, share;   // flat tiles
    int first, cnt;        // flat index of sequence b's first tile, and how many it has
    int b, nrt, nt, tlo;   // row tiles, token tiles, first token tile of the sequence
    Kv8Seq s;
    Seg seg;
};

// Tiles of a sequence; at least one per row tile, whatever its length.
template <int RT>
__device__ __forceinline__ int seq_tiles(const AttendParams& p, const Kv8Seq& s, int& nrt, int& nt, int& tlo)
{
    nrt = (s.n * p.G + RT - 1) / RT;
    const int have = (int)min((long long)max(s.len, 0), (long long)p.w.max_pages << p.w.lgP);
    const int first = max(s.len, 0) - s.n;  // position of the first row
    tlo = p.window && first >= p.window ? (first - p.window + 1) / kTile : 0;
    nt = max((have + kTile - 1) / kTile - tlo, 1);
    return p.w.KV * nrt * nt;
}

// The segment at pos, which lies in sequence b or behind it.
template <int RT>
__device__ __forceinline__ void walk_enter(const AttendParams& p, Walk& k)
{
    if (k.pos >= k.end) {
        k.seg.t1 = k.seg.t0 = 0;
        return;
    }
#pragma unroll 1
    while (k.pos >= k.first + k.cnt) {
        k.first += k.cnt;
        ++k.b;
        k.s = kv8_seq(p.w, k.b);
        k.cnt = seq_tiles<RT>(p, k.s, k.nrt, k.nt, k.tlo);
    }
    const unsigned local = k.pos - k.first, item = local / k.nt, t = local - item * k.nt;
    k.seg.h = item / k.nrt;
    k.seg.rt = item - k.seg.h * k.nrt;
    k.seg.row0 = k.s.row0, k.seg.n = k.s.n, k.seg.len = k.s.len;
    k.seg.t0 = k.tlo + t;
    k.seg.t1 = min(k.tlo + k.nt, k.seg.t0 + (k.end - k.pos));
    const unsigned item0 = k.pos - t;
    k.seg.c0 = item0 / k.share;
    k.seg.c1 = (item0 + k.nt - 1) / k.share;
}

// a / b of small non-negative numbers by the approximate reciprocal: with
// a < 2^21 its error is less than the half that is added.
__device__ __forceinline__ int quotient(int a, int b)
{
    if (a >= 1 << 21) return a / b;
    return (int)__fdividef((float)a + 0.5f, (float)b);
}

// This CTA's part of the work and its first segment.  Two ways to share it out:
//   by row tiles, where there are no more of them than CTAs and their lengths
//   differ little: a row tile has `per` CTAs, each with one run of its tiles
//   (at least sqrt(nt/12): a part costs the join about a twelfth of a tile.  With
//   a third, one sequence of 16,384 tokens takes 19.8 us instead of 18.7 and one
//   of 131,072 40.9 instead of 35.6; with a 48th, 16.8 and 35.7, but one of 4096
//   14.7 instead of 12.4);
//   by tiles, else: equal runs of the flat list of all tiles.
// Lane l looks at the sequences 32 i + l.
template <int RT>
__device__ __forceinline__ void walk_begin(const AttendParams& p, Walk& k)
{
    const int lane = threadIdx.x & 31, ctas = gridDim.x, me = blockIdx.x;
    int tiles = 0, items = 0, longest = 0;
    constexpr int kKept = 4;
    int nts[kKept], its[kKept];  // of the first 128 sequences, read at once and kept
    // (Faults are reported when a sequence's turn comes, not here: nothing may
    // stand between these loads.)
    auto load = [&](int b0, int& n, int& len) {
        const int b = b0 + lane;
        n = len = 0;
        if (b >= p.w.B) return;
        const int slot = p.w.slot ? p.w.slot[b] : b;
        n = p.w.start ? min(max(p.w.start[b + 1] - p.w.start[b], 0), p.w.max_rows) : p.w.max_rows;
        if (slot >= 0 && slot < p.w.slots) len = p.w.lens[slot];
    };
    auto look = [&](int n, int len, int& nt, int& it) {
        int nrt, tlo;
        Kv8Seq s;
        s.n = n, s.len = len;
        seq_tiles<RT>(p, s, nrt, nt, tlo);
        it = p.w.KV * nrt;
    };
    auto add = [&](int nt, int it) {
        tiles += nt * it;
        items += it;
        longest = max(longest, it ? nt : 0);
    };
    {
        int n[kKept], len[kKept];
#pragma unroll
        for (int i = 0; i < kKept; ++i) load(32 * i, n[i], len[i]);
#pragma unroll
        for (int i = 0; i < kKept; ++i) {
            look(n[i], len[i], nts[i], its[i]);
            add(nts[i], its[i]);
        }
    }
#pragma unroll 1
    for (int b0 = 32 * kKept; b0 < p.w.B; b0 += 32) {
        int n, len, nt, it;
        load(b0, n, len);
        look(n, len, nt, it);
        add(nt, it);
    }
    tiles = __reduce_add_sync(~0u, tiles);
    items = __reduce_add_sync(~0u, items);
    longest = __reduce_max_sync(~0u, longest);
    const int per = items > 0 && items <= ctas ? quotient(ctas, items) : 0;
    const bool by_items = per > 0 && (float)longest <= per * ((float)tiles / ctas + kSlack + 1);
    if (by_items) {
        k.pos = quotient(me, per);
        k.end = items;
    } else {
        k.share = (tiles + ctas - 1) / ctas;
        k.pos = (int)min((long long)k.share * me, (long long)tiles);
        k.end = min(k.pos + k.share, tiles);
    }
    k.first = k.cnt = 0;
    k.b = -1;
    // The 32 sequences that pos lies in, and the one of them.
#pragma unroll 1
    for (int b0 = 0; k.pos < k.end; b0 += 32) {
        int nt = nts[0], it = its[0];
#pragma unroll
        for (int i = 1; i < kKept; ++i)
            if (b0 == 32 * i) nt = nts[i], it = its[i];
        if (b0 >= 32 * kKept) {
            int n, len;
            load(b0, n, len);
            look(n, len, nt, it);
        }
        const int c = by_items ? it : nt * it;
        int x = c;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(~0u, x, d);
            if (lane >= d) x += y;
        }
        const unsigned past = __ballot_sync(~0u, k.first + x > k.pos);
        if (past) {
            const int l = __ffs(past) - 1;
            k.b = b0 + l - 1;  // walk_enter reads the sequence itself
            k.first += __shfl_sync(~0u, x - c, l);
            break;
        }
        k.first += __shfl_sync(~0u, x, 31);
    }
    if (by_items && k.pos < k.end) {
        // Row tile `pos` as a list of its own: walk_enter sees the tiles of the
        // part, no others.
        const int part = me - k.pos * per;
        ++k.b;
        k.s = kv8_seq(p.w, k.b);
        seq_tiles<RT>(p, k.s, k.nrt, k.nt, k.tlo);
        const int item = k.pos - k.first;
        const int run = max(quotient(k.nt + per - 1, per), (int)ceilf(sqrtf((float)k.nt * (1.0f / 12.0f))));
        k.seg.h = quotient(item, k.nrt);
        k.seg.rt = item - k.seg.h * k.nrt;
        k.seg.row0 = k.s.row0, k.seg.n = k.s.n, k.seg.len = k.s.len;
        k.seg.t0 = min(part * run, k.nt) + k.tlo;
        k.seg.t1 = min(part * run + run, k.nt) + k.tlo;
        k.seg.c0 = k.pos * per;
        k.seg.c1 = k.seg.c0 + quotient(k.nt + run - 1, run) - 1;
        k.pos = k.end = 0;  // and no more after it
        return;
    }
    walk_enter<RT>(p, k);
}

template <int RT>
__device__ __forceinline__ void walk_next(const AttendParams& p, Walk& k)
{
    k.pos += k.seg.t1 - k.seg.t0;
    walk_enter<RT>(p, k);
}

// ------------------------------------------------------------- shared memory --

constexpr int kDigits = 3;  // of queries and weights

template <int RT>
struct Shape {
    static constexpr int N = (kDigits * RT + 15) / 16 * 16;
    static constexpr uint32_t kPBytes = N * 128;
};

struct Bars {
    uint64_t kfull[kMaxStages], kempty[kMaxStages], vfull[kMaxStages], vempty[kMaxStages];
    uint64_t sfull[2], sempty[2], pfull[2], ofull[2], joined[2];
    uint64_t mfull[kMeta], segfull[kMeta], qfull, jdone, jlast;
};

struct Meta {
    float ks[4], vs[4];
    int valid;  // bit j: page j of the tile exists
    int pad[3];
};

template <int RT>
struct alignas(16) Small {
    float stat_max[2][4][RT];  // per softmax warp: its page's maximum
    float stat_sum[2][4][RT];  // and the sum of its 32 (bits of 1 + weight), an unsigned integer
    float wmax[2][4][RT];
    float qscale[2][RT];  // by the segment's parity
    int pos[2][RT];
    float join[4][5][RT];      // per join warp: the factor of what was there, then of each page
    float stat_vs[2][4];  // and its page's scale of v
    Meta meta[kMeta];
    Seg seg[kMeta];
    Bars bars;
    uint32_t tmem;
    int abort;
    int last;
    int kfills[kMaxStages], vfills[kMaxStages];
};

template <int RT>
__device__ __forceinline__ void store_rows(float* dst, const float (&x)[RT])
{
#pragma unroll
    for (int r = 0; r < RT; r += 4)
        *reinterpret_cast<float4*>(dst + r) = make_float4(x[r], x[r + 1], x[r + 2], x[r + 3]);
}

template <int N>
__device__ __forceinline__ void load_rows(const float* src, float (&x)[N])
{
#pragma unroll
    for (int r = 0; r < N; r += 4) {
        const float4 v = *reinterpret_cast<const float4*>(src + r);
        x[r] = v.x, x[r + 1] = v.y, x[r + 2] = v.z, x[r + 3] = v.w;
    }
}

// Value of column r's digits.  A digit's sum over 128 products is below 2^22 in
// magnitude, so two of them make one int32.  Conversions are slow here (they
// share a quarter-rate pipe with ex2): the third digit takes 1.5 * 2^23 in its
// integer, which is a float's bit pattern.
template <int C>
__device__ __forceinline__ float digits_value(const int (&c)[kDigits][C], int r)
{
    const float hi = (float)(c[0][r] * 256 + c[1][r]);
    return fmaf(hi, 256.0f, __int_as_float(0x4b400000 + c[2][r]) - 12582912.0f);
}

template <typename T, int RT, int HDW>
__global__ void __launch_bounds__(kThreads, 2) k_kv8_attend(const __grid_constant__ AttendParams p)
{
    constexpr int N = Shape<RT>::N;
    constexpr uint32_t kStage = kTile * HDW, kPBytes = Shape<RT>::kPBytes;
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
    const int P = p.w.P, lgP = p.w.lgP, NP = kTile >> lgP;
    auto over_g = [&](int f) { return (int)__umulhi((unsigned)f, p.inv_g) + (p.G == 1 ? f : 0); };

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
            mbar_init(&br.ofull[i], 1);
            mbar_init(&br.joined[i], 4);
        }
        for (int i = 0; i < kMeta; ++i) {
            mbar_init(&br.mfull[i], 1);
            mbar_init(&br.segfull[i], 1);
        }
        mbar_init(&br.qfull, 4);
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
    // The other warps' view of the walk: the next segment, once it is known.
    // The ring cannot overrun: the copies are at most kMaxStages tiles ahead of
    // the products, these 2 ahead of the softmax and that 2 ahead of the join.
    int seg_at = 0;
    auto next_seg = [&](Seg& k) -> bool {
        const int i = seg_at % kMeta;
        if (!warp_wait(&br.segfull[i], seg_at / kMeta & 1, err, abort)) return false;
        k = z.seg[i];
        ++seg_at;
        return k.t1 > k.t0;
    };

    uint64_t* last_bar = nullptr;  // of the product issued last
    int last_ph = 0;
    if (warp == 8) {
        // ---------------------------------------------------------- copies --
        // Page entries come in batches of up to 32 pages of one segment, one
        // per lane, each fetched while the batch before it is copied.
        int st = 0, use = 0, mt = 0;
        struct Batch {
            int tiles, unit, have;
        };
        Walk k;
        walk_begin<RT>(p, k);
        auto publish = [&]() {
            if (lane == 0) {
                z.seg[seg_at % kMeta] = k.seg;
                mbar_arrive(&br.segfull[seg_at % kMeta]);
            }
            ++seg_at;
        };
        publish();
        int at_t = k.seg.t0;
        auto fetch = [&]() -> Batch {
            Batch f{0, 0, 0};
            if (at_t == k.seg.t1) {  // (at the end: t1 = t0, and so on)
                if (k.seg.t1 == k.seg.t0) return f;
                walk_next<RT>(p, k);
                publish();
                at_t = k.seg.t0;
            }
            f.tiles = min(k.seg.t1 - at_t, 32 / NP);
            if (f.tiles == 0) return f;
            const int pg = at_t * NP + lane;
            if (lane < f.tiles * NP && (long long)pg << p.w.lgP < k.s.len) {
                const int x = kv8_unit(p.w, k.s, pg, k.seg.h);
                if (x >= 0) f.have = 1, f.unit = x;
            }
            at_t += f.tiles;
            return f;
        };
        Batch nxt = fetch();
        bool ok = true;
        while (ok && nxt.tiles) {
            const Batch cur = nxt;
            float ks = 0.0f, vs = 0.0f;  // of this lane's page
            for (int i = 0; ok && i < cur.tiles; ++i) {
                const int at = i * NP, j = lane - at;
                if (use > 0 && !(ok = warp_wait(&br.kempty[st], (use - 1) & 1, err, abort))) break;
                const bool mine = lane >= at && lane < at + NP;
                if (lane == at) {
                    z.kfills[st] += 1;
                    mbar_arrive_expect_tx(&br.kfull[st], kStage);
                }
                __syncwarp();
                if (mine) tma_page(&p.kmap, ksm + st * kStage + j * P * HDW, cur.unit, &br.kfull[st]);
                if (i == 0) {
                    // The batch's scales, and the next batch's entries, are on
                    // their way while the first tile is.
                    if (cur.have) ks = p.w.ks[cur.unit], vs = p.w.vs[cur.unit];
                    nxt = fetch();
                }
                if (use > 0 && !(ok = warp_wait(&br.vempty[st], (use - 1) & 1, err, abort))) break;
                if (lane == at) {
                    z.vfills[st] += 1;
                    mbar_arrive_expect_tx(&br.vfull[st], kStage);
                }
                __syncwarp();
                if (mine) tma_page(&p.vmap, vsm + st * kStage + j * P * HDW, cur.unit, &br.vfull[st]);
                Meta& m = z.meta[mt];
                const unsigned valid = __ballot_sync(~0u, mine && cur.have) >> at;
                if (mine) m.ks[j] = ks, m.vs[j] = vs;
                if (lane == at) m.valid = (int)valid;
                __syncwarp();
                if (lane == at) mbar_arrive(&br.mfull[mt]);
                if (++st == S) st = 0, ++use;
                if (++mt == kMeta) mt = 0;
            }
        }
    } else if (warp == 9) {
        // ------------------------------------------------------------ MMAs --
        const uint32_t idS = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (8u << 24);
        const uint32_t idO = (2u << 4) | (1u << 7) | (1u << 15) | ((uint32_t)(N >> 3) << 17) | (8u << 24);
        int kst = 0, kuse = 0, vst = 0, vuse = 0, sb = 0, su = 0, pb = 0, pu = 0, ob = 0, ou = 0, seg = 0, tile = 0;
        // An address moves a descriptor by its sixteenth.
        const uint64_t qd = desc_of(sptr(qsm), 8 * HDW, kSw), kd = desc_of(sptr(ksm), 8 * HDW, kSw);
        const uint64_t vd = desc_of(sptr(vsm), 8 * HDW, kSw), pd = desc_of(sptr(psm), 1024, 2u);
        const int lg_per = lgP - 5, first_of = (1 << lg_per) - 1;
        auto issue_s = [&](bool fresh) -> bool {
            if (fresh && !warp_wait(&br.qfull, seg++ & 1, err, abort)) return false;
            if (!warp_wait(&br.kfull[kst], kuse & 1, err, abort)) return false;
            if (su > 0 && !warp_wait(&br.sempty[sb], (su - 1) & 1, err, abort)) return false;
            fence_after();
            if (elect()) {
#pragma unroll
                for (int i = 0; i < HDW / 32; ++i)
                    mma_i8(tm_s + sb * N, kd + (uint32_t)(kst * (kStage / 16) + 2 * i), qd + 2 * i, idS, i > 0);
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
            // The outputs' buffer: of the tile before the last, or of the last.
            if (p.nO == 2 ? pu > 0 : tile > 0) {
                const int of = p.nO == 2 ? tile - 2 : tile - 1;
                if (!warp_wait(&br.joined[of & 1], of >> 1 & 1, err, abort)) return false;
            }
            fence_after();
            if (elect()) {
#pragma unroll
                for (int i = 0; i < kTile / 32; ++i)  // 32 tokens each
                    mma_i8(tm_o + (ob * NP + (i >> lg_per)) * N, vd + (uint32_t)(vst * (kStage / 16) + 2 * HDW * i),
                           pd + (uint32_t)(pb * (kPBytes / 16) + 2 * i), idO, (i & first_of) > 0);
                mma_commit(&br.ofull[ob]);
                mma_commit(&br.vempty[vst]);
            }
            __syncwarp();
            last_bar = &br.ofull[ob], last_ph = ou & 1;
            if (++vst == S) vst = 0, ++vuse;
            if (++pb == 2) pb = 0, ++pu;
            if (++ob == p.nO) ob = 0, ++ou;
            ++tile;
            return true;
        };
        Seg k;
        bool more = next_seg(k), ok = !more || issue_s(true);
        while (ok && more) {
            const int t1 = k.t1;
            for (int t = k.t0; ok && t < t1; ++t) {
                // The next scores first, unless their keys are still on the way:
                // then this tile's outputs, which free its values' stage.
                const bool first = t + 1 < t1 && __all_sync(~0u, mbar_try_wait(&br.kfull[kst], kuse & 1));
                if (first) ok = issue_s(false);
                ok = ok && issue_o();
                if (!first && t + 1 < t1) ok = ok && issue_s(false);
            }
            if (!ok || !(more = next_seg(k))) break;
            ok = issue_s(true);
        }
    } else if (warp < 4) {
        // --------------------------------------------------------- softmax --
        const int tid = threadIdx.x, page = tid >> p.w.lgP;
        int sb = 0, su = 0, pb = 0, pu = 0, mt = 0, mu = 0, seg = 0;
        const uint32_t tm = tm_s + ((uint32_t)warp << 21);
        constexpr float kQMax = 8323072.0f;  // 127 * 256^2
        // Query rows warp, warp + 4, ... of a row tile; lane l has 4 elements.
        constexpr int kRows = RT / 4;
        auto load_q = [&](const Seg& k, float (&x)[kRows][4]) {
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const int f = k.rt * RT + 4 * i + warp, qi = over_g(f), g = f - qi * p.G, e = lane * 4;
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i][j] = 0.0f;
                if (qi >= k.n || e >= p.w.hd) continue;
                const size_t off = (size_t)(k.row0 + qi) * p.ldq + (size_t)(k.h * p.G + g) * p.w.hd + e;
                load4<T>(static_cast<const T*>(p.q) + off, p.vec, x[i]);
            }
        };
        float qx[kRows][4];
        Seg k;
        // Whether all warps of the page say so.  A named barrier costs a tenth of
        // an mbarrier's round trip (25 and 300 cycles), but its wait has no
        // limit: these warps therefore meet the same number of times whatever
        // happens, and leave their loops together, on its answer.
        auto all_of = [&](bool mine) -> bool {
            if (lgP == 5) return mine;
            uint32_t all;
            asm volatile(
                "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %3, 0;\n\t"
                "bar.red.and.pred p, %1, %2, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                : "=r"(all)
                : "r"(lgP == 6 ? 1 + (warp >> 1) : 1), "r"(lgP == 6 ? 64 : 128), "r"((uint32_t)mine)
                : "memory");
            return all != 0;
        };
        bool ok = true, more = all_of(next_seg(k));
        if (more) load_q(k, qx);
        while (more) {
            // The row tile's query rows as digits.  Its last product has read
            // the old ones (its scores have arrived).
            const int base_pos = k.len - k.n, sg = seg & 1;
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const int r = 4 * i + warp, e = lane * 4;
                const float* x = qx[i];
                const float top = warp_max_nan(max_nan(max_nan(fabsf(x[0]), fabsf(x[1])), max_nan(fabsf(x[2]), fabsf(x[3]))));
                const bool fine = top <= 3.402823466e38f;
                // The largest power of two that keeps the row's largest element
                // in range.  Below 3e-32 (no power of two for it) rows count as 0.
                float inv = 0.0f, step = 0.0f;
                if (fine && top > 3e-32f) {
                    const int ex = 252 + 8 * kDigits - (int)(__float_as_uint(top) >> 23);
                    inv = __uint_as_float((uint32_t)ex << 23);
                    if (top * inv > kQMax) inv *= 0.5f;
                    step = 1.0f / inv;
                }
                uint32_t dig[3] = {0, 0, 0};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    int v = fine ? __float2int_rn(x[j] * inv) : 0;
#pragma unroll
                    for (int d = kDigits - 1; d >= 0; --d) {
                        const int lo = (int)(int8_t)v;
                        dig[d] |= (uint32_t)(lo & 255) << (8 * j);
                        v = (v - lo) >> 8;
                    }
                }
                if (e < HDW) {
#pragma unroll
                    for (int d = 0; d < kDigits; ++d) {
                        const int n = d * RT + r;
                        const int sw = HDW == 128 ? (n & 7) : ((n >> 1) & 3);
                        *reinterpret_cast<uint32_t*>(qsm + n * HDW + ((((e >> 4) ^ sw) << 4) | (e & 15))) = dig[d];
                    }
                }
                if (lane == 0) {
                    z.qscale[sg][r] = fine ? step * p.scale2 : __int_as_float(0x7fffffff);
                    z.pos[sg][r] = base_pos + over_g(k.rt * RT + r);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&br.qfull);
            if (!(ok = all_of(warp_wait(&br.qfull, seg++ & 1, err, abort)))) break;
            const int pos_lo = z.pos[sg][0], pos_hi = z.pos[sg][RT - 1];

            const int t0 = k.t0, t1 = k.t1;
#pragma unroll 1
            for (int t = t0; t < t1; ++t) {
                if (t + 1 == t1) {  // the next row tile's rows come during the last tile
                    more = next_seg(k);
                    if (more) load_q(k, qx);
                }
                ok = ok && warp_wait(&br.mfull[mt], mu & 1, err, abort) && warp_wait(&br.sfull[sb], su & 1, err, abort);
                if (lgP == 5 && !ok) break;
                const Meta& m = z.meta[mt];
                const float ks = m.ks[page];
                const int valid = m.valid;
                fence_after();
                float x[RT], mx[RT];
#pragma unroll
                for (int r0 = 0; r0 < RT; r0 += (RT < 8 ? RT : 8)) {
                    constexpr int C = RT < 8 ? RT : 8;
                    int c[kDigits][C];
#pragma unroll
                    for (int d = 0; d < kDigits; ++d) {
                        if constexpr (C == 8) tmem_ld8(tm + sb * N + d * RT + r0, c[d]);
                        else tmem_ld4(tm + sb * N + d * RT + r0, c[d]);
                    }
                    float qs[C];
                    load_rows<C>(&z.qscale[sg][r0], qs);
                    tmem_wait();
#pragma unroll
                    for (int r = 0; r < C; ++r) x[r0 + r] = digits_value<C>(c, r) * (qs[r] * ks);
                }
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&br.sempty[sb]);
                const int tok = t * kTile + tid;
                if (t * kTile + kTile - 1 > pos_lo || valid != (1 << NP) - 1 ||
                    (p.window && pos_hi >= p.window && t * kTile <= pos_hi - p.window)) {
                    const bool there = (valid >> page) & 1;
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const int q = z.pos[sg][r];
                        const bool seen = there && tok <= q && (!p.window || tok > q - p.window);
                        x[r] = seen ? x[r] : -INFINITY;
                    }
                }
#pragma unroll
                for (int r = 0; r < RT; ++r) mx[r] = warp_max_nan(x[r]);
                if (lgP > 5) {  // the page spans several warps
                    const int wn = 1 << (lgP - 5);
                    if (lane == 0) store_rows<RT>(z.wmax[pb][warp], mx);
                    if (!(ok = all_of(ok))) break;
#pragma unroll
                    for (int i = 1; i < 4; ++i) {
                        if (i >= wn) break;
                        const float* other = z.wmax[pb][(warp & ~(wn - 1)) | ((warp + i) & (wn - 1))];
                        float v[RT];
                        load_rows<RT>(other, v);
#pragma unroll
                        for (int r = 0; r < RT; ++r) mx[r] = max_nan(mx[r], v[r]);
                    }
                }
                // The tile before the last is joined: its weights were used and
                // its maxima read.
                // (A warp that gave up here says so at its next all_of.)
                if (pu > 0) ok = warp_wait(&br.joined[pb], (pu - 1) & 1, err, abort);
                float sum[RT];
                uint8_t* pt = psm + pb * kPBytes + (tid & 15);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    // Weight of the token relative to its page's largest: 1 + w
                    // holds it to 23 bits in its low bits.
                    const float ref = mx[r] == -INFINITY ? 0.0f : mx[r];
                    const uint32_t u = __float_as_uint(1.0f + ex2(x[r] - ref));
                    auto put = [&](int n, uint32_t v) { pt[n * 128 + (((tid >> 4) ^ (n & 7)) << 4)] = (uint8_t)v; };
                    put(r, (u >> 16) - 0x80);
                    put(r + RT, u >> 8);
                    put(r + 2 * RT, u);
                    // u - 0x3f800000 per lane
                    sum[r] = __uint_as_float(__reduce_add_sync(~0u, u));
                }
                if (lane == 0) {
                    store_rows<RT>(z.stat_sum[pb][warp], sum);
                    store_rows<RT>(z.stat_max[pb][warp], mx);
                    z.stat_vs[pb][warp] = m.vs[page];
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&br.pfull[pb]);
                if (++sb == p.nS) sb = 0, ++su;
                if (++pb == 2) pb = 0, ++pu;
                if (++mt == kMeta) mt = 0, ++mu;
            }
            more = all_of(more && ok);
        }
    } else if (warp < 8) {
        // ------------------------------------------------------------ join --
        const int tid = threadIdx.x - 128, w4 = warp - 4;
        const uint32_t tm = tm_o + ((uint32_t)w4 << 21);
        int sb = 0, su = 0, ob = 0, ou = 0, meets = 0;
        bool ok = true;
        constexpr float kUnit = 1.0f / 8388608.0f;
        constexpr size_t kPart = RT * 130;
        constexpr int kSets = RT <= 8 ? 1 : RT / 8, kSet = RT < 8 ? RT : 8;
        const int me = blockIdx.x;
        T* out = static_cast<T*>(p.out);
        // Offsets of the row tile's rows, in lane r that of row r (-1: no such
        // row); element `e` of a row from there.
        auto row_of = [&](const Seg& k, long long& off, long long& lse) {
            const int f = k.rt * RT + (lane & (RT - 1)), qi = over_g(f), hq = k.h * p.G + f - qi * p.G;
            const long long row = k.row0 + qi;
            off = qi < k.n ? row * p.ldo + (long long)hq * p.w.hd : -1;
            lse = row * p.H + hq;
        };
        auto lse_of = [&](float m, float l) {
            return m == -INFINITY ? m : (m + log2f(l)) * 0.693147180559945f;
        };
        // Counts this CTA in; true in all join threads if it is the last of n,
        // and then the others' parts can be read.
        auto last_of = [&](int* counter, int n, bool& last) -> bool {
            // The barrier orders the join threads' parts before the counting
            // (release, cumulative), the counting the others' before the reads.
            __syncwarp();
            if (lane == 0) mbar_arrive(&br.jdone);
            if (tid == 0 && mbar_wait_bounded(&br.jdone, meets & 1, err, abort)) {
                int old;
                asm volatile("atom.add.acq_rel.gpu.s32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
                z.last = old == n - 1;
                if (z.last) *counter = 0;
                mbar_arrive(&br.jlast);
            }
            __syncwarp();
            if (!warp_wait(&br.jlast, meets++ & 1, err, abort)) return false;
            last = z.last;
            return true;
        };
        // Row tiles that this CTA shares with others: the one it came into and
        // the one it leaves.
        Seg shared0{}, shared1{};
        int n_shared = 0;
        Seg k;
        while (ok && next_seg(k)) {
            float o[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) o[r] = 0.0f;
            // Lane 8 w + r has softmax warp w's part of rows r, 8 + r, ...
            float m_run[kSets], l_run[kSets];
#pragma unroll
            for (int i = 0; i < kSets; ++i) m_run[i] = -INFINITY, l_run[i] = 0.0f;
            for (int t = k.t0; t < k.t1; ++t) {
                if (!(ok = warp_wait(&br.pfull[sb], su & 1, err, abort))) break;
                const int from = lane >> 3;
                const float vs = z.stat_vs[sb][from];
#pragma unroll
                for (int i = 0; i < kSets; ++i) {
                    const int r = 8 * i + (lane & (kSet - 1));
                    const float mp = z.stat_max[sb][from][r];
                    const float sum = (float)(__float_as_uint(z.stat_sum[sb][from][r]) - 32u * 0x3f800000u);
                    float mn = max_nan(m_run[i], mp);
                    mn = max_nan(mn, __shfl_xor_sync(~0u, mn, 8));
                    mn = max_nan(mn, __shfl_xor_sync(~0u, mn, 16));
                    const float ref = mn == -INFINITY ? 0.0f : mn, f = ex2(mp - ref), a = ex2(m_run[i] - ref);
                    float l = sum * kUnit * f;
                    l += __shfl_xor_sync(~0u, l, 8);
                    l += __shfl_xor_sync(~0u, l, 16);
                    l_run[i] = fmaf(l_run[i], a, l);
                    m_run[i] = mn;
                    if ((lane & 7) < kSet) {
                        if (lane < 8) z.join[w4][0][r] = a;
                        // A page that is masked altogether counts nothing, whatever its scale.
                        if ((from & ((1 << (lgP - 5)) - 1)) == 0)
                            z.join[w4][1 + (from >> (lgP - 5))][r] = mp == -INFINITY ? 0.0f : f * kUnit * vs;
                    }
                }
                __syncwarp();
                if (!(ok = warp_wait(&br.ofull[ob], ou & 1, err, abort))) break;
                fence_after();
                {
                    float w[RT];
                    load_rows<RT>(z.join[w4][0], w);
#pragma unroll
                    for (int r = 0; r < RT; ++r) o[r] *= w[r];
                }
                for (int j = 0; j < NP; ++j) {
#pragma unroll
                    for (int r0 = 0; r0 < RT; r0 += (RT < 8 ? RT : 8)) {
                        constexpr int C = RT < 8 ? RT : 8;
                        int c[kDigits][C];
#pragma unroll
                        for (int d = 0; d < kDigits; ++d) {
                            if constexpr (C == 8) tmem_ld8(tm + (ob * NP + j) * N + d * RT + r0, c[d]);
                            else tmem_ld4(tm + (ob * NP + j) * N + d * RT + r0, c[d]);
                        }
                        float w[C];
                        load_rows<C>(&z.join[w4][1 + j][r0], w);
                        tmem_wait();
#pragma unroll
                        for (int r = 0; r < C; ++r) {
                            o[r0 + r] = fmaf(digits_value<C>(c, r), w[r], o[r0 + r]);
                        }
                    }
                }
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&br.joined[sb]);
                if (++sb == 2) sb = 0, ++su;
                if (++ob == p.nO) ob = 0, ++ou;
            }
            if (!ok) break;
            // Lane r: row r.
            float m_row = m_run[0], l_row = l_run[0];
#pragma unroll
            for (int i = 1; i < kSets; ++i) {
                const float m = __shfl_sync(~0u, m_run[i], lane & 7), l = __shfl_sync(~0u, l_run[i], lane & 7);
                if (lane >> 3 == i) m_row = m, l_row = l;
            }
            if (k.c0 == k.c1) {
                long long off, at;
                row_of(k, off, at);
                const float inv = m_row == -INFINITY ? 0.0f : 1.0f / l_row;  // nothing seen: o is 0
                if (p.lse && w4 == 0 && lane < RT && off >= 0) p.lse[at] = lse_of(m_row, l_row);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const long long to = __shfl_sync(~0u, off, r);
                    const float v = o[r] * __shfl_sync(~0u, inv, r);
                    if (to >= 0 && tid < p.w.hd) out[to + tid] = from_f<T>(v);
                }
            } else {
                // A part: o[RT][128], m[RT], l[RT].
                float* part = p.part + (2 * (size_t)me + (me == k.c0 ? 1 : 0)) * kPart;
#pragma unroll
                for (int r = 0; r < RT; ++r) part[r * 128 + tid] = o[r];
                if (w4 == 0 && lane < RT) part[RT * 128 + lane] = m_row, part[RT * 129 + lane] = l_row;
                if (n_shared++) shared1 = k;
                else shared0 = k;
            }
        }
        // Joins the n <= 32 parts at base, base + stride, ... (the first of them
        // one part further when `shift`), 8 rows at a time: 16 threads have a
        // row, 8 elements each, and lanes j of them weigh the parts j and 16 + j.
        // To another part, or (null) to the output.
        auto join_parts = [&](const float* base, int n, size_t stride, bool shift, float* to, const Seg& k) {
            long long off, at;
            row_of(k, off, at);
            const int j = tid & 15, head = lane & 16;
#pragma unroll 1
            for (int r0 = 0; r0 < RT; r0 += 8) {
                const int r = min(r0 + (tid >> 4), RT - 1);
                const float* row = base + (shift ? kPart : 0);  // of part 0; the others lie one part lower
                auto part_at = [&](int i) { return i ? base + i * stride : row; };
                float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
                const float* mine = part_at(j) + RT * 128 + r;
                if (j < n) m0 = __ldcg(mine), l0 = __ldcg(mine + RT);
                if (16 + j < n) m1 = __ldcg(base + (16 + j) * stride + RT * 128 + r), l1 = __ldcg(base + (16 + j) * stride + RT * 129 + r);
                float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f), b = a;
                float top = max_nan(m0, m1);
#pragma unroll
                for (int d = 8; d; d >>= 1) top = max_nan(top, __shfl_xor_sync(~0u, top, d));
                const float ref = top == -INFINITY ? 0.0f : top, f0 = ex2(m0 - ref), f1 = ex2(m1 - ref);
                float l = fmaf(l0, f0, l1 * f1);
#pragma unroll
                for (int d = 8; d; d >>= 1) l += __shfl_xor_sync(~0u, l, d);
#pragma unroll 4
                for (int i = 0; i < n; ++i) {
                    const float4* v = reinterpret_cast<const float4*>(part_at(i) + r * 128 + j * 8);
                    const float4 x = __ldcg(v), y = __ldcg(v + 1);
                    const float g = __shfl_sync(~0u, i < 16 ? f0 : f1, head | (i & 15));
                    a.x = fmaf(x.x, g, a.x), a.y = fmaf(x.y, g, a.y), a.z = fmaf(x.z, g, a.z), a.w = fmaf(x.w, g, a.w);
                    b.x = fmaf(y.x, g, b.x), b.y = fmaf(y.y, g, b.y), b.z = fmaf(y.z, g, b.z), b.w = fmaf(y.w, g, b.w);
                }
                const long long o_at = __shfl_sync(~0u, off, r), l_at = __shfl_sync(~0u, at, r);
                if (r0 + (tid >> 4) >= RT) continue;
                if (to) {
                    float4* t = reinterpret_cast<float4*>(to + r * 128 + j * 8);
                    t[0] = a, t[1] = b;
                    if (j == 0) to[RT * 128 + r] = top, to[RT * 129 + r] = l;
                } else if (o_at >= 0) {
                    const float inv = top == -INFINITY ? 0.0f : 1.0f / l;
                    const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (j * 8 + e < p.w.hd) out[o_at + j * 8 + e] = from_f<T>(v[e] * inv);
                    if (p.lse && j == 0) p.lse[l_at] = lse_of(top, l);
                }
            }
        };
        // Shared row tiles: whoever comes last joins them, in token order.
#pragma unroll 1
        for (int i = 0; ok && i < n_shared; ++i) {
            const Seg q = i ? shared1 : shared0;
            bool last = false;
            const int g0 = join_group(q.c0, me);
            const bool grouped = join_grouped(q.c0, q.c1);
#pragma unroll 1
            for (int step = join_first(q.c0, q.c1, me); step < 2; ++step) {
                const JoinStep s = join_step(step, q.c0, q.c1, me);
                if (!(ok = last_of(p.counters + s.counter, s.n, last)) || !last) break;
                const bool shift = step || g0 == q.c0;
                const float* base = p.part + 2 * (size_t)(step ? q.c0 : g0) * kPart;
                const size_t stride = 2 * kPart * (step && grouped ? kJoinGroup : 1);
                join_parts(base, s.n, stride, shift, step ? nullptr : const_cast<float*>(base) + (shift ? kPart : 0), q);
            }
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

// Rows of a row tile: a sequence's rows (tokens x query heads of a KV head) if
// they fit, else 16.  32 measured slower (64-token chunks 83 us against 67, 512
// tokens 320 against 265): its registers leave one CTA per SM.
int pick_rt(const quantr_kv8_batch* b, int G)
{
    const long long rows = (long long)b->max_rows * G;
    return rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
}

struct Plan {
    int stages, nS, nO, cols, grid;
    size_t smem;
};

template <int RT, int HDW>
Plan make_plan(int lgP)
{
    constexpr int N = Shape<RT>::N;
    static_assert(N * (1 + kTile / 32) <= 256, "half of an SM's TMEM holds a buffer of either");
    const int NP = kTile >> lgP;
    Plan r{};
    // Two buffers of scores and of outputs where 256 TMEM columns hold them, half
    // an SM's (two CTAs per SM); else one of outputs, else one of either (rows of
    // 16 over pages of 32: 64-token chunks 53 us, 70 with one CTA per SM and two
    // buffers of scores).
    const int tries[3][2] = {{2, 2}, {2, 1}, {1, 1}};
    for (auto& t : tries) {
        r.nS = t[0], r.nO = t[1];
        r.cols = 32;
        while (r.cols < N * (t[0] + t[1] * NP)) r.cols *= 2;
        if (r.cols <= 256) break;
    }
    const size_t fixed = 1024 + 2 * Shape<RT>::kPBytes + N * HDW + sizeof(Small<RT>);
    const size_t room = 113 * 1024;
    r.stages = (int)std::min<size_t>(kMaxStages, (room - fixed) / (2 * kTile * HDW));
    r.smem = fixed + (size_t)r.stages * 2 * kTile * HDW;
    r.grid = std::min(2 * device_sm_count(), kJoinCtas);
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

template <typename T, int RT, int HDW>
cudaError_t run(AttendParams& p, const quantr_kv8_pool* pool, void* ws, const LaunchCfg& c)
{
    const Plan r = make_plan<RT, HDW>(p.w.lgP);
    static int configured = -1;
    cudaError_t e = ensure_smem_attr(k_kv8_attend<T, RT, HDW>, 227 * 1024, configured);
    if (e != cudaSuccess) return e;
    if (!encode_map(&p.kmap, pool->k, pool, HDW) || !encode_map(&p.vmap, pool->v, pool, HDW))
        return cudaErrorNotSupported;
    p.stages = r.stages, p.nS = r.nS, p.nO = r.nO, p.tmem_cols = r.cols;
    p.counters = static_cast<int*>(ws);
    p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + 4096);
    return launch_ex(k_kv8_attend<T, RT, HDW>, dim3(r.grid), kThreads, r.smem, c, p);
}

template <typename T, int HDW>
cudaError_t run_rt(int rt, AttendParams& p, const quantr_kv8_pool* pool, void* ws, const LaunchCfg& c)
{
    switch (rt) {
    case 4: return run<T, 4, HDW>(p, pool, ws, c);
    case 8: return run<T, 8, HDW>(p, pool, ws, c);
    default: return run<T, 16, HDW>(p, pool, ws, c);
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
    if ((rc = kv8_check_rows(out, ldo, need, type)) || (rc = kv8_check_rows(q, ldq, need, type))) return rc;
    if (!kv8_aligned({lse})) return QUANTR_ERR_BAD_ARG;
    if (!workspace || ((uintptr_t)workspace & 255) ||
        workspace_bytes < quantr_kv8_attend_workspace_bytes(pool, batch, n_heads, max_len))
        return QUANTR_ERR_WORKSPACE;
    const int rt = pick_rt(batch, n_heads / pool->n_kv_heads);
    {  // flat tile numbers and f * G (above) are 32-bit
        const double G = n_heads / pool->n_kv_heads, rows = (double)batch->max_rows * G + rt;
        const double tiles = (double)tables->max_pages * pool->page_tokens / kTile + 1;
        if (rows * G >= 4294967296.0 || (double)batch->B * pool->n_kv_heads * (rows / rt + 1) * tiles >= 2147483648.0)
            return QUANTR_ERR_TOO_LARGE;
    }
    AttendParams p{};
    p.w = kv8_view(pool, tables, batch, layer);
    p.q = q, p.out = out, p.lse = lse, p.ldq = ldq, p.ldo = ldo;
    p.vec = type == QUANTR_TYPE_F32 ? aligned(q, ldq, 4, 16) : aligned(q, ldq, 2, 8);
    p.H = n_heads, p.G = n_heads / pool->n_kv_heads;
    // A window past every position hides nothing.
    p.window = window < (long long)tables->max_pages * pool->page_tokens ? window : 0;
    p.inv_g = p.G == 1 ? 0 : (unsigned)(((1ull << 32) + p.G - 1) / p.G);
    p.scale2 = (float)((double)scale * 1.4426950408889634);
    LaunchCfg c;
    c.stream = (cudaStream_t)stream;
    const cudaError_t e = with_type(type, [&](auto* t) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
        return pool->head_dim <= 64 ? run_rt<T, 64>(rt, p, pool, workspace, c) : run_rt<T, 128>(rt, p, pool, workspace, c);
    });
    return kv8_done(e);
}

} // extern "C"
