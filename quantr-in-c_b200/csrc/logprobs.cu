// logprobs.cu -- log probabilities of given tokens, entropy and the k largest
// alternatives of rows of logits (public contract: include/quantr_cuda.h).
//
// Mathematics.  With c = log2(e)/temperature every thread keeps the running
// maximum m of its logits, s = sum 2^(c(x-m)) and e = sum 2^(c(x-m)) c(x-m);
// joined over the row,
//   lse = m/temperature + ln s,  entropy = ln2 (log2 s - e/s).
// One pass: each logit is read once, whatever is asked for.
//
// Alternatives cost the pass nothing but a store: a thread keeps the maximum of
// each group of its elements, which the softmax needs anyway.  Then a threshold
// that k elements reach at least (each warp's ceil(k/8)-th largest thread
// maximum, the least of the 8 warps), and only the groups that reach it are
// read again, a few dozen of thousands.  Their elements are ranked as 64-bit
// keys (logit, ~id), all different: ties go to the lower id, and the order of
// the threads does not matter.  More than a buffer of them (a row of equal
// values) are ranked by k passes instead.
#include "kv8.cuh"

#include <algorithm>
#include <cmath>

namespace qr {
namespace {

constexpr int kLpThreads = 256, kLpWarps = kLpThreads / 32;
constexpr int kVecs = 4;          // 16-byte loads per thread and tile
constexpr int kMaxTop = 64;
constexpr int kGroups = 32;       // groups of a thread's tiles, at most
constexpr int kHits = 1024;       // groups that are read again
constexpr int kCap = 1024;        // candidates that are ranked against each other
constexpr int kMaxMerge = kCap;   // candidates that the last CTA of a row merges

typedef unsigned long long u64;

struct LpArgs {
    const void* x;
    long long ldl;
    int rows, V, k, split;
    float inv_t, c;  // 1/temperature, and times log2(e)
    const int* token;
    float* logprob;
    float* entropy;
    float* lse;
    int* top_id;
    float* top_lp;
    int* counters;  // one per row, zero between calls
    float4* part;   // (m, s, e) of every (row, slice)
    u64* keys;      // k of every (row, slice)
};

// Order of alternatives: larger logits first, then lower ids.  0 is below all
// (-inf and NaN are not alternatives).
__device__ __forceinline__ u64 lp_key(float x, int id)
{
    if (!(x > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(x + 0.0f);  // -0 is 0
    const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (u64)o << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float lp_value(u64 key)
{
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

__device__ __forceinline__ float lp_ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lp_max_nan(float a, float b)
{
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// Largest of the warp's values (NaN counts as none).
__device__ __forceinline__ float warp_max(float x)
{
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

struct Sums {
    float m, s, e;
};

// Both about the larger maximum.
__device__ __forceinline__ Sums join(Sums a, Sums b, float c)
{
    Sums r;
    r.m = fmaxf(a.m, b.m);
    if (r.m == -INFINITY) return {r.m, a.s + b.s, a.e + b.e};
    const float da = (a.m - r.m) * c, db = (b.m - r.m) * c;
    const float fa = lp_ex2(da), fb = lp_ex2(db);
    r.s = a.s * fa + b.s * fb;
    r.e = (a.m == -INFINITY ? a.s : fmaf(a.s, da, a.e) * fa) + (b.m == -INFINITY ? b.s : fmaf(b.s, db, b.e) * fb);
    return r;
}

template <typename T>
struct Vec {
    static constexpr int n = 16 / sizeof(T);
};

// Elements of one 16-byte load.
template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float* x)
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            x[i] = __uint_as_float(w[i]);
        } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}

// The largest element of one load (NaN counts as none).
template <typename T>
__device__ __forceinline__ float vec_max(const uint4& v)
{
    if constexpr (sizeof(T) == 4) {
        return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)),
                     fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
    } else if constexpr (std::is_same_v<T, __half>) {
        const __half2* h = reinterpret_cast<const __half2*>(&v);
        const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return fmaxf(__low2float(m), __high2float(m));
    } else {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
        const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return fmaxf(__low2float(m), __high2float(m));
    }
}

struct LpShared {
    u64 buf[kCap];
    u64 tops[kMaxTop];
    u64 best[kLpWarps];
    float low[kLpWarps];
    int count, hits, last;
    Sums sums[kLpWarps];
    uint16_t hit[kHits];  // group * threads + thread
    float group_max[1];  // [group][thread]
};

// The k largest of the buffer's n keys to z.tops, in order (0 where there are
// fewer).  All threads.
__device__ __forceinline__ void rank_keys(LpShared& z, int n, int k)
{
    for (int i = threadIdx.x; i < k; i += kLpThreads)
        if (i >= n) z.tops[i] = 0;
    for (int i = threadIdx.x; i < n; i += kLpThreads) {
        const u64 key = z.buf[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) rank += z.buf[j] > key || (z.buf[j] == key && j < i);  // 0 may repeat
        if (rank < k) z.tops[rank] = key;
    }
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads, 4) k_logprobs(const LpArgs a)
{
    constexpr int VE = Vec<T>::n;
    extern __shared__ __align__(16) uint8_t raw[];
    LpShared& z = *reinterpret_cast<LpShared*>(raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) z.count = z.hits = 0;
    pdl_wait();
    const int row = blockIdx.x / a.split, slice = blockIdx.x % a.split;
    const T* x = static_cast<const T*>(a.x) + row * a.ldl;
    // Elements before the first 16-byte boundary, whole vectors, the rest.
    const int head = min(a.V, (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)));
    const int nvec = (a.V - head) / VE, tail = a.V - head - nvec * VE;
    const int per = (nvec + a.split - 1) / a.split, v0 = min(nvec, slice * per), v1 = min(nvec, v0 + per);
    const uint4* xv = reinterpret_cast<const uint4*>(x + head);
    const bool ends = (head | tail) && slice == a.split - 1;  // the last slice takes the ragged ends too
    const int tiles = (v1 - v0 + kVecs * kLpThreads - 1) / (kVecs * kLpThreads) + (ends ? 1 : 0);
    const int whole = tiles - (ends ? 1 : 0);
    const uint32_t ninf = sizeof(T) == 4 ? 0xff800000u : std::is_same_v<T, __half> ? 0xfc00fc00u : 0xff80ff80u;
    const uint4 none = make_uint4(ninf, ninf, ninf, ninf);

    Sums st{-INFINITY, 0.0f, 0.0f};
    // Tiles of a group: as few as keep the groups within kGroups.
    const int gt = (tiles + kGroups - 1) / kGroups;
    float gmax = -INFINITY;
    int left = gt, group = 0;
    uint4 nxt[kVecs];
    auto fetch = [&](int t) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const int v = v0 + (t * kVecs + i) * kLpThreads + tid;
            nxt[i] = t < whole && v < v1 ? __ldcs(xv + v) : none;
        }
    };
    fetch(0);
    for (int t = 0; t < tiles; ++t) {
        uint4 cur[kVecs];
#pragma unroll
        for (int i = 0; i < kVecs; ++i) cur[i] = nxt[i];
        fetch(t + 1);
        const bool ragged = t == whole;  // one element per thread: head, then tail
        float extra = -INFINITY;
        if (ragged && tid < head + tail) extra = to_f<T>(x[tid < head ? tid : a.V - tail + (tid - head)]);
        float mt = extra;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) mt = fmaxf(mt, vec_max<T>(cur[i]));
        if (mt > st.m) {
            if (st.m > -INFINITY) {
                const float d = (st.m - mt) * a.c, r = lp_ex2(d);
                st.e = fmaf(st.s, d, st.e) * r;
                st.s *= r;
            }
            st.m = mt;
        }
        const float ref = st.m == -INFINITY ? 0.0f : st.m * a.c;
        float s0 = 0.0f, s1 = 0.0f, e0 = 0.0f, e1 = 0.0f;
        if (fabsf(ref) <= 3.402823466e38f && !ragged) {
#pragma unroll
            for (int v = 0; v < kVecs; ++v) {
                float f[VE];
                unpack<T>(cur[v], f);
#pragma unroll
                for (int i = 0; i < VE; i += 2) {
                    // 2^-200 is 0; the bound keeps -inf out of 0 * -inf and NaN in.
                    const float d0 = lp_max_nan(fmaf(f[i], a.c, -ref), -200.0f);
                    const float d1 = lp_max_nan(fmaf(f[i + 1], a.c, -ref), -200.0f);
                    const float p0 = lp_ex2(d0), p1 = lp_ex2(d1);
                    s0 += p0, s1 += p1;
                    e0 = fmaf(p0, d0, e0), e1 = fmaf(p1, d1, e1);
                }
            }
        } else {
            // The ragged ends, and maxima so large that c times them has no
            // float (a row of nothing but the type's lowest value, say).
            const float base = st.m == -INFINITY ? 0.0f : st.m;
            auto one = [&](float y) {
                const float d = lp_max_nan((y - base) * a.c, -200.0f), p = lp_ex2(d);
                s0 += p;
                e0 = fmaf(p, d, e0);
            };
            one(extra);
#pragma unroll 1
            for (int v = 0; v < kVecs; ++v) {
                float f[VE];
                unpack<T>(v == 0 ? cur[0] : v == 1 ? cur[1] : v == 2 ? cur[2] : cur[3], f);
#pragma unroll
                for (int i = 0; i < VE; ++i) one(f[i]);
            }
        }
        st.s += s0 + s1;
        st.e += e0 + e1;

        gmax = fmaxf(gmax, mt);
        if (--left == 0) {
            if (a.k) z.group_max[group * kLpThreads + tid] = gmax;
            gmax = -INFINITY, left = gt, ++group;
        }
    }
    if (a.k) {
        if (left < gt) z.group_max[group++ * kLpThreads + tid] = gmax;
        // A threshold that at least k elements of the slice reach, if there are
        // k above -inf at all.
        float mine = st.m, low = -INFINITY;
        for (int i = (a.k + kLpWarps - 1) / kLpWarps; i; --i) {
            low = warp_max(mine);
            const unsigned who = __ballot_sync(~0u, mine == low);
            if (lane == __ffs(who) - 1) mine = -INFINITY;
        }
        if (lane == 0) z.low[warp] = low;
        __syncthreads();
        low = z.low[0];
        for (int w = 1; w < kLpWarps; ++w) low = fminf(low, z.low[w]);
        // Calls g with the keys of vector i (of kVecs * gt) of a group's thread.
        auto keys_of = [&](int q, int th, int i, auto&& g) {
            const int t = q * gt + i / kVecs;
            if (t == whole && ends && i % kVecs == 0) {
                if (th >= head + tail) return;
                const int id = th < head ? th : a.V - tail + (th - head);
                const float y = to_f<T>(x[id]);
                if (y >= low) g(lp_key(y, id));
            } else if (t < whole) {
                const int v = v0 + (t * kVecs + i % kVecs) * kLpThreads + th;
                if (v >= v1) return;
                float f[VE];
                unpack<T>(xv[v], f);
#pragma unroll
                for (int j = 0; j < VE; ++j)
                    if (f[j] >= low) g(lp_key(f[j], head + v * VE + j));
            }
        };
        if (st.m >= low && st.m > -INFINITY)
            for (int q = 0; q < group; ++q)
                if (z.group_max[q * kLpThreads + tid] >= low) {
                    const int at = atomicAdd(&z.hits, 1);
                    if (at < kHits) z.hit[at] = (uint16_t)(q * kLpThreads + tid);
                }
        __syncthreads();
        const int hits = z.hits;
        if (hits <= kHits)
            for (int i = tid; i < hits * kVecs * gt; i += kLpThreads) {
                const int h = z.hit[i / (kVecs * gt)];
                keys_of(h / kLpThreads, h % kLpThreads, i % (kVecs * gt), [&](u64 key) {
                    if (!key) return;
                    const int at = atomicAdd(&z.count, 1);
                    if (at < kCap) z.buf[at] = key;
                });
            }
        __syncthreads();
        const int n = z.count;
        if (hits <= kHits && n <= kCap) {
            rank_keys(z, n, a.k);
        } else {
            u64 last = ~0ull;
            for (int i = 0; i < a.k; ++i) {
                u64 best = 0;
                for (int q = 0; q < group; ++q)
                    if (z.group_max[q * kLpThreads + tid] >= low)
                        for (int j = 0; j < kVecs * gt; ++j)
                            keys_of(q, tid, j, [&](u64 key) {
                                if (key < last && key > best) best = key;
                            });
                for (int d = 16; d; d >>= 1) best = max(best, __shfl_xor_sync(~0u, best, d));
                if (lane == 0) z.best[warp] = best;
                __syncthreads();
                for (int w = 0; w < kLpWarps; ++w) best = max(best, z.best[w]);
                __syncthreads();
                if (tid == 0) z.tops[i] = best;
                last = best;
            }
            __syncthreads();
        }
    }
    // The row's sums: over the warp, the CTA, the slices.
    for (int d = 16; d; d >>= 1) {
        Sums o;
        o.m = __shfl_xor_sync(~0u, st.m, d);
        o.s = __shfl_xor_sync(~0u, st.s, d);
        o.e = __shfl_xor_sync(~0u, st.e, d);
        st = lane & d ? join(o, st, a.c) : join(st, o, a.c);  // the same operands in the same order on both lanes
    }
    if (lane == 0) z.sums[warp] = st;
    __syncthreads();
    st = z.sums[0];
    for (int w = 1; w < kLpWarps; ++w) st = join(st, z.sums[w], a.c);

    if (a.split > 1) {
        const size_t at = (size_t)row * a.split;
        if (tid == 0) a.part[at + slice] = make_float4(st.m, st.s, st.e, 0.0f);
        for (int i = tid; i < a.k; i += kLpThreads) a.keys[(at + slice) * a.k + i] = z.tops[i];
        __threadfence();
        __syncthreads();
        if (tid == 0) {
            z.last = atomicAdd(a.counters + row, 1) == a.split - 1;
            if (z.last) a.counters[row] = 0;
            __threadfence();
        }
        __syncthreads();
        if (!z.last) return;
        st = {-INFINITY, 0.0f, 0.0f};
        for (int i = 0; i < a.split; ++i) {
            const float4 q = __ldcg(a.part + at + i);
            st = join(st, Sums{q.x, q.y, q.z}, a.c);
        }
        if (a.k) {
            for (int i = tid; i < a.split * a.k; i += kLpThreads) z.buf[i] = __ldcg(a.keys + at * a.k + i);
            __syncthreads();
            rank_keys(z, a.split * a.k, a.k);
        }
    }
    constexpr float ln2 = 0.693147180559945f;
    const float l2 = log2f(st.s);
    const bool bad = st.s != st.s || st.m == INFINITY;
    float lse = fmaf(l2, ln2, st.m * a.inv_t), ent = (l2 - st.e / st.s) * ln2;
    if (st.m == -INFINITY) lse = -INFINITY, ent = 0.0f;
    if (bad) lse = ent = NAN;
    if (tid == 0) {
        if (a.lse) a.lse[row] = lse;
        if (a.entropy) a.entropy[row] = ent;
        if (a.logprob) {
            const int t = a.token[row];
            float lp = 0.0f;
            if (t >= 0 && t < a.V) lp = lse == -INFINITY ? -INFINITY : to_f<T>(x[t]) * a.inv_t - lse;
            else if (t != -1) lp = NAN;
            a.logprob[row] = lp;
        }
    }
    for (int i = tid; i < a.k; i += kLpThreads) {
        const u64 key = z.tops[i];
        if (a.top_id) a.top_id[(size_t)row * a.k + i] = key ? (int)~(uint32_t)key : -1;
        if (a.top_lp) a.top_lp[(size_t)row * a.k + i] = bad ? NAN : key ? lp_value(key) * a.inv_t - lse : -INFINITY;
    }
}

// Slices per row.  One CTA streams about 9 KB per microsecond and SM while 4 of
// them share an SM; a slice is at least two tiles.
int lp_split(int rows, int vocab, int k)
{
    const long long slots = 4ll * device_sm_count();
    const int most = std::max(1, std::min((vocab + 8191) / 8192, k ? kMaxMerge / k : 1024));
    if ((long long)rows * most <= slots) return most;
    if (rows < slots) return std::max(1, (int)(slots / rows));
    // Several waves: the split whose last wave is fullest.
    int best = 1;
    double fill = 0.0;
    for (int s = 1; s <= std::min(most, 8); ++s) {
        const long long n = (long long)rows * s, waves = (n + slots - 1) / slots;
        const double f = (double)n / (waves * slots) - 0.01 * s;
        if (f > fill) fill = f, best = s;
    }
    return best;
}

struct LpWs {
    size_t part, keys, total;
};
LpWs lp_ws(int rows, int split, int k)
{
    LpWs w;
    w.part = ((size_t)rows * 4 + 255) & ~size_t(255);
    w.keys = w.part + (size_t)rows * split * sizeof(float4);
    w.total = w.keys + (size_t)rows * split * k * sizeof(u64);
    return w;
}

} // namespace
} // namespace qr

extern "C" {

using namespace qr;

size_t quantr_logprobs_workspace_bytes(int rows, int vocab, int k)
{
    if (rows <= 0 || vocab <= 0 || k < 0 || k > kMaxTop) return 256;
    return std::max<size_t>(256, lp_ws(rows, lp_split(rows, vocab, k), k).total);
}

int quantr_logprobs_dev(const void* x, long long ldl, uint32_t type, int rows, int vocab, float temperature,
                        const int* token, float* logprob, float* entropy, float* lse, int k, int* top_id,
                        float* top_logprob, void* workspace, size_t workspace_bytes, void* stream)
{
    if (!kv8_float_type(type)) return QUANTR_ERR_UNSUPPORTED_TYPE;
    if (rows < 0 || vocab <= 0 || k < 0 || ldl < vocab || !(temperature > 0.0f) || !std::isfinite(temperature) ||
        !std::isfinite(1.0f / temperature))
        return QUANTR_ERR_BAD_ARG;
    if (k > kMaxTop) return QUANTR_ERR_TOO_LARGE;
    if (rows == 0) return QUANTR_OK;
    if (!x || (uintptr_t)x % (type == QUANTR_TYPE_F32 ? 4 : 2) || (logprob && !token)) return QUANTR_ERR_BAD_ARG;
    if (!workspace || ((uintptr_t)workspace & 255) ||
        workspace_bytes < quantr_logprobs_workspace_bytes(rows, vocab, k))
        return QUANTR_ERR_WORKSPACE;
    LpArgs a{};
    a.x = x, a.ldl = ldl, a.rows = rows, a.V = vocab, a.k = k, a.split = lp_split(rows, vocab, k);
    if ((long long)rows * a.split > 0x7fffffffll) return QUANTR_ERR_TOO_LARGE;
    a.inv_t = (float)(1.0 / (double)temperature);
    a.c = (float)(1.4426950408889634 / (double)temperature);
    a.token = token, a.logprob = logprob, a.entropy = entropy, a.lse = lse, a.top_id = top_id, a.top_lp = top_logprob;
    const LpWs w = lp_ws(rows, a.split, k);
    uint8_t* base = static_cast<uint8_t*>(workspace);
    a.counters = reinterpret_cast<int*>(base);
    a.part = reinterpret_cast<float4*>(base + w.part);
    a.keys = reinterpret_cast<u64*>(base + w.keys);
    LaunchCfg c;
    c.stream = (cudaStream_t)stream;
    return kv8_done(with_type(type, [&](auto* t) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
        // Tiles of the longest slice, with one for the ragged ends.
        const int vecs = vocab / Vec<T>::n, per = (vecs + a.split - 1) / a.split;
        const int tiles = (per + kVecs * kLpThreads - 1) / (kVecs * kLpThreads) + 1;
        const size_t smem = sizeof(LpShared) + (k ? std::min(tiles, kGroups) * kLpThreads * sizeof(float) : 0);
        return launch_ex(k_logprobs<T>, dim3((unsigned)(rows * a.split)), kLpThreads, smem, c, a);
    }));
}

} // extern "C"
