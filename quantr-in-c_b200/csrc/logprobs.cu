// logprobs.cu -- log probabilities of given tokens, entropy and the k largest
// alternatives of rows of logits (public contract: include/quantr_cuda.h).
//
// Mathematics.  With c = log2(e)/temperature every thread keeps the running
// maximum m of its logits, s = sum 2^(c(x-m)) and e = sum 2^(c(x-m)) c(x-m);
// joined over the row,
//   lse = m/temperature + ln s,  entropy = ln2 (log2 s - e/s).
// A thread's exponents are c x - r with r = c m rounded, one instruction for two;
// what the rounding leaves out (lo = c m - r) is part of its sums, and taken out
// of them where they meet sums about another maximum.  Where lo would be large
// (maxima millions of temperatures from 0) they are c (x - m).
// One pass: each logit is read once, whatever is asked for.
//
// Alternatives cost the pass nothing but a store: a thread keeps the maximum of
// each group of its elements, which the softmax needs anyway.  Then a threshold
// that k elements of the row reach at least (the k-th largest of every warp's
// few largest thread maxima), and only the groups that reach it are read again,
// about k of thousands.  Their elements are ranked as 64-bit keys (logit, ~id), all
// different: ties go to the lower id, and the order of the threads does not
// matter.
//
// A row is one CTA, or a cluster of up to 8 where there are few rows, joined
// through distributed shared memory.
//
// What bounds it, and what it measured (B200, 6.54 TB/s copy): 2047 rows of
// 151,936 bf16 logits (622 MB), 4 alternatives: 123 us, 5.1 TB/s; without them 106
// (an ex2 per logit beside the conversions, and 3.46 waves of CTAs); 1024 fp32
// rows without them, the same bytes, 95, 6.5 TB/s: memory.  64 fp32 rows (39 MB),
// 20 alternatives: 15.0 us; 10.8 without: a row's end is a chain of a threshold, a
// second read and a ranking.  One row of 32,000: 6.4 to 6.6 us, 3.4 without
// alternatives: latency.
// Tried and not kept: rings of bulk copies in shared memory (without
// alternatives 146 -> 187 us at that step), CTAs that stay and fetch the next row
// during a row's end (no change), 128 threads per CTA (prompt 123 -> 145).
#include "kv8.cuh"

#include <algorithm>
#include <cmath>

namespace qr {
namespace {

constexpr int kLpThreads = 256, kLpWarps = kLpThreads / 32;
constexpr int kVecs = 4;          // 16-byte loads per thread and tile
constexpr int kMaxTop = 64;
constexpr int kGroups = 32;       // groups of a thread's tiles, at most
constexpr int kMaxHeads = 128;    // values that the threshold is chosen from
constexpr int kHits = 1024;       // groups that are read again
constexpr int kCap = 512;         // candidates that are ranked against each other
constexpr int kMaxSplit = 8;      // CTAs of a row: one cluster

typedef unsigned long long u64;

struct LpArgs {
    const void* x;
    long long ldl;
    int V, k, split;
    double inv_t;  // 1 / temperature
    float c;       // times log2(e)
    // Maxima m (above < m, |m| <= most) for which a tile's exponents are
    // c x - (c m rounded), one instruction each: that rounding is then half a unit
    // at most, and Low<T>::bound weighs nothing beside m.
    float above, most;
    const int* token;
    float* logprob;
    float* entropy;
    float* lse;
    int* top_id;
    float* top_lp;
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

// A thread's sums are about 2^(c m - lo): see `take`.
struct Sums {
    float m, s, e, lo;
};

// Sums of more than one thread are held in 64 bits: a row's rounding is then
// that of its results, for a few operations per row.
struct WideSums {
    float m;
    double s, e;
};

// The warp's sums about their largest maximum; in all lanes.  `lo`: see Sums.
__device__ __forceinline__ WideSums join_warp(WideSums a, float c, float lo = 0.0f)
{
    const float m = warp_max(a.m);
    if (m > -INFINITY) {
        // (2^-200 is 0, and bounded it makes no 0 * -inf; NaN stays.)
        const float d = lp_max_nan((a.m - m) * c - lo, -200.0f), f = lp_ex2(d);
        a.e = (a.e + a.s * d) * f;
        a.s *= f;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        a.s += __shfl_xor_sync(~0u, a.s, d);
        a.e += __shfl_xor_sync(~0u, a.e, d);
    }
    a.m = m;
    return a;
}

template <typename T>
struct Vec {
    static constexpr int n = 16 / sizeof(T);
};

// Two floats that one instruction works on (fma/add.rn.f32x2).
struct F2 {
    u64 v;
};
__device__ __forceinline__ F2 f2(float a, float b)
{
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void f2_get(F2 x, float& a, float& b)
{
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v));
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c)
{
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ F2 f2_add(F2 a, F2 b)
{
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

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

// The bound below which the fast path takes logits as one: 2^-200 of the
// maximum or less, so that their weight is 0 either way, and -inf makes no
// 0 * -inf.
template <typename T>
struct Low {
    static constexpr float bound = -1e30f;
};
template <>
struct Low<__half> {
    static constexpr float bound = -65504.0f;
};

// The same elements, not below the bound; NaN stays NaN.
template <typename T>
__device__ __forceinline__ void unpack_bounded(const uint4& v, float* x)
{
    if constexpr (sizeof(T) == 4) {
        unpack<T>(v, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = lp_max_nan(x[i], Low<T>::bound);
    } else {
        uint4 u = v;
        uint32_t* w = &u.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<T, __half>) {
                const __half2 b = __float2half2_rn(Low<T>::bound);
                const __half2 h = __hmax2_nan(*reinterpret_cast<const __half2*>(&w[i]), b);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 b = __float2bfloat162_rn(Low<T>::bound);
                const __nv_bfloat162 h = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), b);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        unpack<T>(u, x);
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

struct alignas(16) LpShared {
    float heads[kMaxHeads];  // every warp's largest thread maxima, of the whole row
    u64 slot[kCap];          // of the row's first CTA, as are found and part: a stretch for each CTA's candidates
    u64 buf[kCap];
    u64 tops[kMaxTop];
    u64 best[kLpWarps];
    float low;
    WideSums part[kMaxSplit * kLpWarps];
    int found[kMaxSplit];
    int count, hits;
    uint16_t hit[kHits];  // group * threads + thread
    float group_max[1];   // [group][thread]
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
        for (int j = 0; j < n; ++j) rank += z.buf[j] > key;
        if (rank < k) z.tops[rank] = key;
    }
    __syncthreads();
}

// More candidates than the buffer holds: the k best of the row with those above
// `low`, then of those equal to it the first ones; k passes where even the
// former are too many.  By the row's first CTA.
template <typename T>
__device__ __noinline__ void crowded(const LpArgs& a, LpShared& z, const T* x, float low)
{
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __syncthreads();
    if (tid == 0) z.count = 0;
    __syncthreads();
    for (int v = tid; v < a.V; v += kLpThreads) {
        const float y = to_f<T>(x[v]);
        if (!(y > low)) continue;
        const int i = atomicAdd(&z.count, 1);
        if (i < kCap) z.buf[i] = lp_key(y, v);
    }
    __syncthreads();
    int n = z.count;
    if (n <= kCap - kLpThreads) {
        for (int v0 = 0; v0 < a.V && n < a.k && low > -INFINITY; v0 += kLpThreads) {
            const int v = v0 + tid;
            __syncthreads();
            if (v < a.V && to_f<T>(x[v]) == low) z.buf[atomicAdd(&z.count, 1)] = lp_key(low, v);
            __syncthreads();
            n = z.count;
        }
        rank_keys(z, n, a.k);
        return;
    }
    u64 last = ~0ull;
    for (int i = 0; i < a.k; ++i) {
        u64 best = 0;
        for (int v = tid; v < a.V; v += kLpThreads) {
            const u64 key = lp_key(to_f<T>(x[v]), v);
            if (key < last && key > best) best = key;
        }
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

template <typename T>
__global__ void __launch_bounds__(kLpThreads, 4) k_logprobs(const LpArgs a)
{
    constexpr int VE = Vec<T>::n;
    extern __shared__ __align__(16) uint8_t raw[];
    LpShared& z = *reinterpret_cast<LpShared*>(raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) z.count = z.hits = 0, z.low = -INFINITY;
    if (tid < kMaxHeads) z.heads[tid] = -INFINITY;
    if (tid < kMaxSplit * kLpWarps) z.part[tid] = {-INFINITY, 0.0, 0.0};
    cluster_arrive();  // every CTA of the cluster has begun, and zeroed its counts: waited for before the first remote access
    pdl_wait();
    const int row = blockIdx.x / a.split, slice = blockIdx.x % a.split;
    const T* x = static_cast<const T*>(a.x) + row * a.ldl;
    // The given token and its logit, two dependent loads that the pass hides.
    int token = -1;
    float token_x = 0.0f;
    if (tid == 0 && slice == 0 && a.logprob) {
        token = a.token[row];
        if (token >= 0 && token < a.V) token_x = to_f<T>(x[token]);
    }
    // Elements before the first 16-byte boundary, whole vectors, the rest.
    const int head = min(a.V, (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)));
    const int nvec = (a.V - head) / VE, tail = a.V - head - nvec * VE;
    const int per = (nvec + a.split - 1) / a.split, v0 = min(nvec, slice * per), v1 = min(nvec, v0 + per);
    const uint4* xv = reinterpret_cast<const uint4*>(x + head);
    const bool ends = (head | tail) && slice == a.split - 1;  // the last slice takes the ragged ends too
    const int full = (v1 - v0) / (kVecs * kLpThreads);        // tiles without a bound to look at
    const int whole = (v1 - v0 + kVecs * kLpThreads - 1) / (kVecs * kLpThreads), tiles = whole + (ends ? 1 : 0);
    const uint32_t ninf = sizeof(T) == 4 ? 0xff800000u : std::is_same_v<T, __half> ? 0xfc00fc00u : 0xff80ff80u;
    const uint4 none = make_uint4(ninf, ninf, ninf, ninf);

    Sums st{-INFINITY, 0.0f, 0.0f, 0.0f};
    // Tiles of a group: as few as keep the groups within kGroups.
    const int gt = (tiles + kGroups - 1) / kGroups;
    float gmax = -INFINITY;
    int left = gt, group = 0;
    const F2 c2 = f2(a.c, a.c);
    bool plain = false;  // see LpArgs
    // The running maximum takes `mt` in; the group's, too.
    auto raise = [&](float mt) {
        if (mt > st.m) {
            plain = mt > a.above && fabsf(mt) <= a.most;
            const float lo = plain ? fmaf(mt, a.c, -(mt * a.c)) : 0.0f;
            if (st.m > -INFINITY) {
                const float d = lp_max_nan((st.m - mt) * a.c + (lo - st.lo), -200.0f), r = lp_ex2(d);
                st.e = fmaf(st.s, d, st.e) * r;
                st.s *= r;
            }
            st.m = mt, st.lo = lo;
        }
        gmax = fmaxf(gmax, mt);
        if (--left == 0) {
            if (a.k) z.group_max[group * kLpThreads + tid] = gmax;
            gmax = -INFINITY, left = gt, ++group;
        }
    };
    auto one = [&](float y) {
        const float base = st.m == -INFINITY ? 0.0f : st.m;
        // 2^-200 is 0; the bound keeps -inf out of 0 * -inf and NaN in.
        const float d = lp_max_nan((y - base) * a.c + st.lo, -200.0f), p = lp_ex2(d);
        st.s += p;
        st.e = fmaf(p, d, st.e);
    };
    auto take = [&](const uint4 (&cur)[kVecs]) {
        float mt = vec_max<T>(cur[0]);
#pragma unroll
        for (int i = 1; i < kVecs; ++i) mt = fmaxf(mt, vec_max<T>(cur[i]));
        raise(mt);
        if (plain) {
            const float ref = -st.m * a.c;
            const F2 r2 = f2(ref, ref);
            F2 s2 = f2(0.0f, 0.0f), e2 = s2;
#pragma unroll
            for (int v = 0; v < kVecs; ++v) {
                float f[VE];
                unpack_bounded<T>(cur[v], f);
#pragma unroll
                for (int i = 0; i < VE; i += 2) {
                    const F2 d = f2_fma(f2(f[i], f[i + 1]), c2, r2);
                    float d0, d1;
                    f2_get(d, d0, d1);
                    const F2 p = f2(lp_ex2(d0), lp_ex2(d1));
                    s2 = f2_add(s2, p);
                    e2 = f2_fma(p, d, e2);
                }
            }
            float x0, x1;
            f2_get(s2, x0, x1);
            st.s += x0 + x1;
            f2_get(e2, x0, x1);
            st.e += x0 + x1;
        } else {
            // Nothing above the bound yet, or a maximum millions of temperatures
            // from 0 (a row of nothing but the type's lowest value, say), whose
            // product with c says nothing about differences: those come first.
#pragma unroll 1
            for (int v = 0; v < kVecs; ++v) {
                float f[VE];
                unpack<T>(v == 0 ? cur[0] : v == 1 ? cur[1] : v == 2 ? cur[2] : cur[3], f);
#pragma unroll
                for (int i = 0; i < VE; ++i) one(f[i]);
            }
        }
    };
    // Two tiles in flight.
    const uint4* at = xv + v0 + tid;
    auto fetch = [&](uint4 (&buf)[kVecs], int t) {
        if (t < full) {
            const uint4* p = at + (size_t)t * (kVecs * kLpThreads);
#pragma unroll
            for (int i = 0; i < kVecs; ++i) buf[i] = __ldcs(p + i * kLpThreads);
        }
    };
    {
        uint4 b0[kVecs], b1[kVecs];
        fetch(b0, 0);
        fetch(b1, 1);
        for (int t = 0; t < full; t += 2) {
            take(b0);
            fetch(b0, t + 2);
            if (t + 1 < full) {
                take(b1);
                fetch(b1, t + 3);
            }
        }
        if (whole > full) {
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                const int v = v0 + (full * kVecs + i) * kLpThreads + tid;
                b0[i] = v < v1 ? __ldcs(xv + v) : none;
            }
            take(b0);
        }
    }
    if (ends) {  // one element per thread: head, then tail
        const float y = tid < head + tail ? to_f<T>(x[tid < head ? tid : a.V - tail + (tid - head)]) : -INFINITY;
        raise(y);
        if (tid < head + tail) one(y);
    }
    // Warps that the threshold looks at: all of them, or those that a short row
    // fills (a split row's slices are long).
    const int nw = a.split > 1 ? kLpWarps : max(1, min(kLpWarps, nvec / 32));
    // Each warp's `per_warp` largest thread maxima, told to every CTA of the row.
    const int heads = nw * a.split, per_warp = a.k ? min((2 * a.k + heads - 1) / heads, min(32, kMaxHeads / heads)) : 0;
    float y = st.m, head_val = -INFINITY;
    if (a.k && left < gt) z.group_max[group++ * kLpThreads + tid] = gmax;
    for (int i = 0; i < per_warp && warp < nw; ++i) {
        const float top = warp_max(y);
        const unsigned who = __ballot_sync(~0u, y == top);
        if (lane == __ffs(who) - 1) y = -INFINITY;
        if (lane == i) head_val = top;
    }
    const WideSums mine = join_warp({st.m, st.s, st.e}, a.c, st.lo);
    cluster_wait();
    if (warp < nw && lane < per_warp)
        for (int r = 0; r < a.split; ++r)
            st_remote(remote_of(&z.heads[(slice * nw + warp) * per_warp + lane], r), head_val);
    if (lane == 0) {
        const uint32_t to = remote_of(&z.part[slice * kLpWarps + warp], 0);
        st_remote(to, mine.m);
        st_remote(to + 8, (u64)__double_as_longlong(mine.s));
        st_remote(to + 16, (u64)__double_as_longlong(mine.e));
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (a.k) {
        // The k-th largest of them, which k of the row's elements reach; none
        // where a short row has fewer.
        const int n = heads * per_warp;
        if (tid < n) {
            const float v = z.heads[tid];
            int above = 0, reach = 0;
#pragma unroll 4
            for (int i = 0; i < n; i += 4) {
                const float4 h = *reinterpret_cast<const float4*>(&z.heads[i]);
                above += (h.x > v) + (h.y > v) + (h.z > v) + (h.w > v);
                reach += (h.x >= v) + (h.y >= v) + (h.z >= v) + (h.w >= v);
            }
            if (above < a.k && a.k <= reach) z.low = v;
        }
        __syncthreads();
        const float low = z.low;
        // Candidates go to this CTA's stretch of the first CTA's slots.
        const int room = kCap / a.split;
        const uint32_t slots = remote_of(&z.slot[slice * room], 0);
        auto push = [&](float y, int id) {
            if (!(y >= low && y > -INFINITY)) return;
            const int i = atomicAdd(&z.count, 1);
            if (i < room) st_remote(slots + 8 * i, lp_key(y, id));
        };
        if (st.m >= low && st.m > -INFINITY)
            for (int q = 0; q < group; ++q)
                if (z.group_max[q * kLpThreads + tid] >= low) {
                    const int i = atomicAdd(&z.hits, 1);
                    if (i < kHits) z.hit[i] = (uint16_t)(q * kLpThreads + tid);
                }
        __syncthreads();
        const int hits = min(z.hits, kHits);
        for (int i = tid; i < hits * kVecs * gt; i += kLpThreads) {
            // Vector i % (kVecs * gt) of the group.
            const int h = z.hit[i / (kVecs * gt)], j = i % (kVecs * gt), th = h % kLpThreads;
            const int t = h / kLpThreads * gt + j / kVecs;
            if (t < whole) {
                const int v = v0 + (t * kVecs + j % kVecs) * kLpThreads + th;
                if (v >= v1) continue;
                float f[VE];
                unpack<T>(xv[v], f);
#pragma unroll
                for (int e = 0; e < VE; ++e) push(f[e], head + v * VE + e);
            } else if (t < tiles && j % kVecs == 0 && th < head + tail) {
                const int id = th < head ? th : a.V - tail + (th - head);
                push(to_f<T>(x[id]), id);
            }
        }
        __syncthreads();
        if (tid == 0) st_remote(remote_of(&z.found[slice], 0), z.hits > kHits || z.count > room ? -1 : z.count);
        __syncwarp();
        cluster_arrive();
        if (slice) return;  // nobody reads this CTA's shared memory any more
        cluster_wait();
        // The stretches, one behind the other: warp r moves CTA r's.
        int total = 0, at = 0;
        bool fits = true;
#pragma unroll
        for (int r = 0; r < kMaxSplit; ++r) {
            const int m = r < a.split ? z.found[r] : 0;
            fits &= m >= 0;
            if (r < warp) at += m;
            total += m;
        }
        if (fits && warp < a.split)
            for (int i = lane; i < z.found[warp]; i += 32) z.buf[at + i] = z.slot[warp * room + i];
        __syncthreads();
        if (fits) rank_keys(z, total, a.k);
        else crowded<T>(a, z, x, low);
    } else if (slice) {
        return;
    }
    // The row's sums, from every warp's (64 places, the others empty), and its
    // results: one warp's work, the others' issue slots are the next row's.
    if (warp) return;
    WideSums sum = z.part[lane];
    if (a.split * kLpWarps > 32) {
        const WideSums u = z.part[32 + lane];
        const bool up = u.m > sum.m;
        const WideSums &hi = up ? u : sum, &lo = up ? sum : u;
        const float d = hi.m > -INFINITY ? lp_max_nan((lo.m - hi.m) * a.c, -200.0f) : 0.0f, f = lp_ex2(d);
        sum = {hi.m, hi.s + lo.s * f, hi.e + (lo.e + lo.s * d) * f};
    }
    sum = join_warp(sum, a.c);
    const double ls = log(sum.s);
    const bool bad = sum.s != sum.s || sum.m == INFINITY;
    double lse = sum.m * a.inv_t + ls, ent = ls - sum.e / sum.s * 0.6931471805599453;
    if (sum.m == -INFINITY) lse = -INFINITY, ent = 0.0;
    if (bad) lse = ent = NAN;
    if (tid == 0) {
        if (a.lse) a.lse[row] = (float)lse;
        if (a.entropy) a.entropy[row] = (float)ent;
        if (a.logprob) {
            double lp = 0.0;
            if (token >= 0 && token < a.V) lp = lse == -INFINITY ? -INFINITY : token_x * a.inv_t - lse;
            else if (token != -1) lp = NAN;
            a.logprob[row] = (float)lp;
        }
    }
    for (int i = lane; i < a.k; i += 32) {
        const u64 key = z.tops[i];
        if (a.top_id) a.top_id[(size_t)row * a.k + i] = key ? (int)~(uint32_t)key : -1;
        if (a.top_lp) a.top_lp[(size_t)row * a.k + i] = bad ? NAN : key ? (float)(lp_value(key) * a.inv_t - lse) : -INFINITY;
    }
}

// CTAs per row: a row has a fixed cost (launch, threshold, ranking), so a row
// is split only while there are fewer CTAs than two per SM.
int lp_split(int rows, int vocab)
{
    const int most = std::min(kMaxSplit, std::max(1, (vocab + 4095) / 4096));
    return std::min(most, (2 * device_sm_count() + rows - 1) / rows);
}

} // namespace
} // namespace qr

extern "C" {

using namespace qr;

size_t quantr_logprobs_workspace_bytes(int rows, int vocab, int k)
{
    (void)rows, (void)vocab, (void)k;
    return 0;
}

int quantr_logprobs_dev(const void* x, long long ldl, uint32_t type, int rows, int vocab, float temperature,
                        const int* token, float* logprob, float* entropy, float* lse, int k, int* top_id,
                        float* top_logprob, void* workspace, size_t workspace_bytes, void* stream)
{
    if (!kv8_float_type(type)) return QUANTR_ERR_UNSUPPORTED_TYPE;
    if (rows < 0 || vocab <= 0 || k < 0 || ldl < vocab || !(temperature > 0.0f) || !std::isfinite(temperature) ||
        !std::isfinite((float)(1.4426950408889634 / (double)temperature)))
        return QUANTR_ERR_BAD_ARG;
    if (k > kMaxTop) return QUANTR_ERR_TOO_LARGE;
    if (rows == 0) return QUANTR_OK;
    if (!x || !kv8_aligned({x}, kv8_type_bytes(type)) || (logprob && !token)) return QUANTR_ERR_BAD_ARG;
    if (!kv8_aligned({token, logprob, entropy, lse, top_id, top_logprob})) return QUANTR_ERR_BAD_ARG;
    (void)workspace, (void)workspace_bytes;
    LpArgs a{};
    a.x = x, a.ldl = ldl, a.V = vocab, a.k = k, a.split = lp_split(rows, vocab);
    if ((long long)rows * a.split > 0x7fffffffll) return QUANTR_ERR_TOO_LARGE;
    a.inv_t = 1.0 / (double)temperature;
    a.c = (float)(1.4426950408889634 / (double)temperature);
    a.token = token, a.logprob = logprob, a.entropy = entropy, a.lse = lse, a.top_id = top_id, a.top_lp = top_logprob;
    LaunchCfg c;
    c.stream = (cudaStream_t)stream;
    return kv8_done(with_type(type, [&](auto* t) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
        a.above = Low<T>::bound + 200.0f / a.c;
        // (None where c times the bound has no float, which would be 0 * -inf.)
        a.most = std::isfinite(Low<T>::bound * a.c) ? 8388608.0f / a.c : -1.0f;
        // Tiles of the longest slice, with one for the ragged ends.
        const int vecs = vocab / Vec<T>::n, per = (vecs + a.split - 1) / a.split;
        const int tiles = (per + kVecs * kLpThreads - 1) / (kVecs * kLpThreads) + 1;
        const size_t smem = sizeof(LpShared) + (k ? std::min(tiles, kGroups) * kLpThreads * sizeof(float) : 0);
        return launch_cluster(k_logprobs<T>, dim3((unsigned)(rows * a.split)), kLpThreads, smem, a.split, c, a);
    }));
}

} // extern "C"
