// kv8.cu -- the 8-bit paged KV cache: writing rows into pages, reading them
// back (public contract: include/quantr_cuda.h).
#include "kv8.cuh"

#include <algorithm>

namespace qr {
namespace {

// ----------------------------------------------------------------- append --

constexpr int kVecs = 4;           // 16-byte vectors of a page that a thread holds
constexpr int kAppendMax = 1024;   // threads: 128 rows of 128 fp32 elements

// Block maximum.
__device__ __forceinline__ uint32_t block_max(uint32_t u, uint32_t* red)
{
    u = __reduce_max_sync(0xffffffffu, u);
    if (blockDim.x == 32) {
        __syncwarp();
        return u;
    }
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = u;
    __syncthreads();
    u = 0;
    for (int i = 0; i < (int)blockDim.x / 32; ++i) u = max(u, red[i]);
    return u;
}

// Magnitudes order like their bits, infinities and NaN above all others: the
// largest of a vector's as an integer of the element's width, and its value
// (NaN for either of those).
template <typename T>
__device__ __forceinline__ uint32_t vec_top(const uint4& v, uint32_t m)
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) m = max(m, w[i] & 0x7fffffffu);
        else m = __vmaxu2(m, w[i] & 0x7fff7fffu);  // two maxima, joined below
    }
    return m;
}
template <typename T>
__device__ __forceinline__ uint32_t top_bits(uint32_t m)
{
    return sizeof(T) == 4 ? m : max(m & 0xffffu, m >> 16);
}
template <typename T>
__device__ __forceinline__ float top_value(uint32_t u)
{
    float f;
    if constexpr (sizeof(T) == 4) f = __uint_as_float(u);
    else if constexpr (std::is_same_v<T, __half>) f = __half2float(__ushort_as_half((unsigned short)u));
    else f = __uint_as_float(u << 16);
    return f <= 3.402823466e38f ? f : __int_as_float(0x7fffffff);
}

// Least j >= 0 with room * 2^j >= top (both finite, room >= 2^-120).
__device__ __forceinline__ int doublings(float top, float room)
{
    if (top <= room) return 0;
    const uint32_t a = __float_as_uint(top), b = __float_as_uint(room);
    return (int)(a >> 23) - (int)(b >> 23) + ((a & 0x7fffffu) > (b & 0x7fffffu) ? 1 : 0);
}

// The rows of a sequence that fall into the m-th page they touch: positions
// lo .. hi-1, the first of them row `row`.
struct PageRows {
    int at, lo, hi;  // page of the sequence
    long long row;
};

__device__ __forceinline__ PageRows page_rows(const Kv8View& w, const Kv8Seq& s, int m)
{
    PageRows r;
    const int first = max(s.len - s.n, 0), skip = max(s.n - s.len, 0);  // rows before position 0 are skipped
    r.at = (first >> w.lgP) + m;
    r.lo = max(r.at << w.lgP, first);
    r.hi = (int)min(((long long)r.at + 1) << w.lgP, (long long)s.len);
    r.row = (long long)s.row0 + skip + (r.lo - first);
    return r;
}

// How the threads of a CTA walk the items of a page's rows, one by one: items of
// a row, and what a step of all threads adds.
struct RowWalk {
    int per_row, drow, dcol;
    uint32_t inv;  // ceil(2^16 / per_row): a thread's row without a division
};

RowWalk row_walk(int per_row, int threads)
{
    return {per_row, threads / per_row, threads % per_row, (65535u + per_row) / per_row};
}

// Row `row` (at p) and item `col` of it that the thread is at.
template <typename T>
struct RowAt {
    T* p;
    int col;
    __device__ __forceinline__ RowAt(const RowWalk& w, T* base, long long ld)
    {
        const int row = (int)(threadIdx.x * w.inv >> 16);
        col = (int)threadIdx.x - row * w.per_row;
        p = base + row * ld;
    }
    __device__ __forceinline__ void step(const RowWalk& w, long long ld, long long dld)
    {
        p += dld;
        col += w.dcol;
        if (col >= w.per_row) col -= w.per_row, p += ld;
    }
};

struct AppendArgs {
    Kv8View w;
    const void* src[2];  // k, v
    long long ld[2];
    int vec[2];
    RowWalk walk;
};

// One CTA per (sequence, page of it that rows fall into, head, k or v): a
// thread holds its vectors of the new rows from the maximum to the codes, so
// the rows are read once, and a chain of three dependent loads (length, page,
// old scale) is all that a single token waits for.  64 sequences' tokens (fp32, 4
// heads of 128): 2.3 us, latency.  8 prompts of up to 2048 tokens (bf16, 46 MB):
// 11.5 us, 3.9 TB/s: that chain, a barrier and the stores one after another, and
// conversions beside them (issue slots 82 % used while a CTA is there).
template <typename T>
__global__ void __launch_bounds__(kAppendMax) k_kv8_append(const AppendArgs a)
{
    constexpr int VE = 16 / sizeof(T);
    __shared__ uint32_t red[kAppendMax / 32];
    pdl_wait();
    const Kv8View& w = a.w;
    const int h = blockIdx.y >> 1, kv = blockIdx.y & 1, threads = blockDim.x;
    const Kv8Seq s = kv8_seq(w, blockIdx.z);
    const PageRows r = page_rows(w, s, blockIdx.x);
    if (r.hi <= r.lo) return;
    const T* src = static_cast<const T*>(a.src[kv]) + r.row * a.ld[kv] + (long long)h * w.hd;
    // The rows' vectors, in order.
    const int n = (r.hi - r.lo) * a.walk.per_row, had = r.lo - (r.at << w.lgP);
    uint4 x[kVecs];
    {
        RowAt<const T> at(a.walk, src, a.ld[kv]);
        const long long dld = a.walk.drow * a.ld[kv];
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            x[i] = make_uint4(0, 0, 0, 0);
            if ((int)threadIdx.x + i * threads < n) {
                const T* p = at.p + at.col * VE;
                if (a.vec[kv]) {
                    x[i] = *reinterpret_cast<const uint4*>(p);
                } else {
                    T* e = reinterpret_cast<T*>(&x[i]);
#pragma unroll
                    for (int j = 0; j < VE; ++j) e[j] = p[j];
                }
            }
            at.step(a.walk, a.ld[kv], dld);
        }
    }
    const int unit = kv8_unit(w, s, r.at, h);
    if (unit < 0) return;
    int8_t* page = (kv ? w.v : w.k) + (size_t)unit * w.P * w.hd;
    float* scale = (kv ? w.vs : w.ks) + unit;
    const float old = had ? *scale : 0.0f;
    uint32_t mb = 0;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) mb = vec_top<T>(x[i], mb);
    const float m = top_value<T>(block_max(top_bits<T>(mb), red));  // also: everybody has read the old scale
    float sc;
    int j = 0;
    if (!had) {
        sc = fmaxf(__fdiv_rn(m, 127.0f), 1.17549435e-38f);
        if (m != m) sc = m;
    } else if (m != m || !(fabsf(old) <= 3.402823466e38f)) {
        sc = __int_as_float(0x7fffffff);
    } else {
        j = doublings(m, __fmul_rn(old, 127.0f));
        sc = old;
        for (int i = 0; i < j; ++i) sc *= 2.0f;
    }
    if (j) {  // the page's old codes, rounded to the doubled scale
        const float f = j < 32 ? 1.0f / (float)(1u << j) : 0.0f;
        for (int g = threadIdx.x; g < had * (w.hd >> 2); g += threads) {
            char4 c = reinterpret_cast<char4*>(page)[g];
            c.x = (signed char)__float2int_rn(c.x * f);
            c.y = (signed char)__float2int_rn(c.y * f);
            c.z = (signed char)__float2int_rn(c.z * f);
            c.w = (signed char)__float2int_rn(c.w * f);
            reinterpret_cast<char4*>(page)[g] = c;
        }
    }
    const float inv = sc == sc ? __fdiv_rn(1.0f, sc) : 0.0f;
    int8_t* dst = page + (size_t)had * w.hd;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int q = threadIdx.x + i * threads;
        if (q >= n) break;
        const T* e = reinterpret_cast<const T*>(&x[i]);
        uint32_t c[VE / 4];
#pragma unroll
        for (int g = 0; g < VE / 4; ++g) {
            // x/s is within 127 (and a few ulp) in magnitude: adding 1.5 * 2^23
            // rounds it half to even into the low byte.
            uint32_t v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                v[k] = __float_as_uint(__fadd_rn(__fmul_rn(to_f<T>(e[4 * g + k]), inv), 12582912.0f));
            c[g] = __byte_perm(__byte_perm(v[0], v[1], 0x0040), __byte_perm(v[2], v[3], 0x0040), 0x5410);
            if (sc != sc) c[g] = 0;
        }
        if constexpr (VE == 4) *reinterpret_cast<uint32_t*>(dst + q * VE) = c[0];
        else *reinterpret_cast<uint2*>(dst + q * VE) = make_uint2(c[0], c[1]);
    }
    if (threadIdx.x == 0) *scale = sc;
}

// ------------------------------------------------------------------- read --

constexpr int kReadThreads = 256;
constexpr int kReadAtOnce = 4;  // groups of eight codes that a thread loads before it stores

struct ReadArgs {
    Kv8View w;
    void* dst[2];
    long long ld[2];
    int vec[2];
    RowWalk walk;
};

// Eight consecutive elements, in one store where the address allows it.
template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, const float (&x)[8])
{
    if (!vec) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = from_f<T>(x[i]);
    } else if constexpr (sizeof(T) == 4) {
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]),
                     "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
                     : "memory");
    } else {
        uint4 v;
        T* t = reinterpret_cast<T*>(&v);
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = from_f<T>(x[i]);
        *reinterpret_cast<uint4*>(p) = v;
    }
}

// One CTA per (sequence, page, head, k or v), like the append; a thread takes
// eight codes at a time.  The same prompts to fp32 (76 MB, most of it written):
// 15.1 us, 5.0 TB/s: memory.  CTA m = 0 of a sequence also zeroes its rows before
// position 0.
template <typename T>
__global__ void __launch_bounds__(kReadThreads) k_kv8_read(const ReadArgs a)
{
    pdl_wait();
    const Kv8View& w = a.w;
    const int h = blockIdx.y >> 1, kv = blockIdx.y & 1, m = blockIdx.x;
    const Kv8Seq s = kv8_seq(w, blockIdx.z);
    const PageRows r = page_rows(w, s, m);
    const long long ld = a.ld[kv], dld = a.walk.drow * ld;
    const bool vec = a.vec[kv];
    T* out = static_cast<T*>(a.dst[kv]) + (long long)h * w.hd;
    if (m == 0 && s.n > s.len) {
        const float zero[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        RowAt<T> at(a.walk, out + s.row0 * ld, ld);
        for (int g = threadIdx.x; g < min(s.n, s.n - s.len) * a.walk.per_row; g += kReadThreads) {
            store8<T>(at.p + at.col * 8, vec, zero);
            at.step(a.walk, ld, dld);
        }
    }
    if (r.hi <= r.lo) return;
    const int unit = kv8_unit(w, s, r.at, h);
    const float sc = unit >= 0 ? (kv ? w.vs : w.ks)[unit] : 0.0f;
    const uint2* page = reinterpret_cast<const uint2*>((kv ? w.v : w.k) + ((size_t)max(unit, 0) * w.P + (r.lo & (w.P - 1))) * w.hd);
    const int n = (r.hi - r.lo) * a.walk.per_row;
    RowAt<T> at(a.walk, out + r.row * ld, ld);
    for (int g0 = threadIdx.x; g0 < n; g0 += kReadAtOnce * kReadThreads) {
        uint2 c[kReadAtOnce];
#pragma unroll
        for (int i = 0; i < kReadAtOnce; ++i) {
            const int g = g0 + i * kReadThreads;
            c[i] = unit >= 0 && g < n ? page[g] : make_uint2(0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < kReadAtOnce; ++i) {
            // The bytes, offset by 128, as the low bits of 2^23.
            const uint32_t u[2] = {c[i].x ^ 0x80808080u, c[i].y ^ 0x80808080u};
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                x[k] = (__uint_as_float(__byte_perm(u[k >> 2], 0x4b000000u, 0x7440 + (k & 3))) - 8388736.0f) * sc;
            if (g0 + i * kReadThreads < n) store8<T>(at.p + at.col * 8, vec, x);
            at.step(a.walk, ld, dld);
        }
    }
}

// Pages that `rows` consecutive rows can touch.
int span_of(const quantr_kv8_pool* p, int rows)
{
    return (int)(((long long)rows + p->page_tokens - 2) / p->page_tokens + 1);
}

} // namespace
} // namespace qr

extern "C" {

using namespace qr;

int quantr_kv8_append_dev(const void* k, long long ldk, const void* v, long long ldv, uint32_t type,
                          const quantr_kv8_pool* pool, const quantr_kv8_tables* tables,
                          const quantr_kv8_batch* batch, int layer, void* stream)
{
    int rc = kv8_check_call(pool, tables, batch, layer, type);
    if (rc || batch->B == 0 || batch->max_rows == 0) return rc;
    const long long need = (long long)pool->n_kv_heads * pool->head_dim;
    if ((rc = kv8_check_rows(k, ldk, need, type)) || (rc = kv8_check_rows(v, ldv, need, type))) return rc;
    AppendArgs a{};
    a.w = kv8_view(pool, tables, batch, layer);
    const int bytes = type == QUANTR_TYPE_F32 ? 4 : 2;
    a.src[0] = k, a.src[1] = v, a.ld[0] = ldk, a.ld[1] = ldv;
    a.vec[0] = aligned(k, ldk, bytes, 16), a.vec[1] = aligned(v, ldv, bytes, 16);
    if (batch->B > 65535 || pool->n_kv_heads > 32767) return QUANTR_ERR_TOO_LARGE;
    // Threads that hold the most rows a page can get, kVecs vectors each.
    const int per_row = pool->head_dim * bytes / 16, vecs = std::min(batch->max_rows, pool->page_tokens) * per_row;
    const int threads = (std::max((vecs + kVecs - 1) / kVecs, std::min(vecs, 64)) + 31) / 32 * 32;
    a.walk = row_walk(per_row, threads);
    LaunchCfg c;
    c.stream = (cudaStream_t)stream;
    return kv8_done(with_type(type, [&](auto* t) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
        return launch_ex(k_kv8_append<T>, dim3(span_of(pool, batch->max_rows), 2 * pool->n_kv_heads, batch->B), threads, 0, c, a);
    }));
}

int quantr_kv8_read_dev(void* k, long long ldk, void* v, long long ldv, uint32_t type, const quantr_kv8_pool* pool,
                        const quantr_kv8_tables* tables, const quantr_kv8_batch* batch, int layer, void* stream)
{
    int rc = kv8_check_call(pool, tables, batch, layer, type);
    if (rc || batch->B == 0 || batch->max_rows == 0) return rc;
    const long long need = (long long)pool->n_kv_heads * pool->head_dim;
    if ((rc = kv8_check_rows(k, ldk, need, type)) || (rc = kv8_check_rows(v, ldv, need, type))) return rc;
    ReadArgs a{};
    a.w = kv8_view(pool, tables, batch, layer);
    const int bytes = type == QUANTR_TYPE_F32 ? 4 : 2;
    a.dst[0] = k, a.dst[1] = v, a.ld[0] = ldk, a.ld[1] = ldv;
    a.vec[0] = aligned(k, ldk, bytes, 8 * bytes), a.vec[1] = aligned(v, ldv, bytes, 8 * bytes);
    if (batch->B > 65535 || pool->n_kv_heads > 32767) return QUANTR_ERR_TOO_LARGE;
    a.walk = row_walk(pool->head_dim / 8, kReadThreads);
    LaunchCfg c;
    c.stream = (cudaStream_t)stream;
    return kv8_done(with_type(type, [&](auto* t) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
        return launch_ex(k_kv8_read<T>, dim3(span_of(pool, batch->max_rows), 2 * pool->n_kv_heads, batch->B), kReadThreads, 0, c, a);
    }));
}

} // extern "C"
