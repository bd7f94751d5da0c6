// kv8.cu -- the 8-bit paged KV cache: writing rows into pages, reading them
// back (public contract: include/quantr_cuda.h).
#include "kv8.cuh"

#include <algorithm>

namespace qr {
namespace {

// ----------------------------------------------------------------- append --

constexpr int kAppendThreads = 256;

// Block maximum of non-negative floats; a NaN or infinity anywhere gives NaN.
__device__ __forceinline__ float block_absmax(float m, bool bad, float* red)
{
    if (bad) m = __int_as_float(0x7fffffff);
    // Non-negative floats (NaN above all) order like their bits.
    uint32_t u = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = __uint_as_float(u);
    __syncthreads();
    u = 0;
    for (int i = 0; i < (int)blockDim.x / 32; ++i) u = max(u, __float_as_uint(red[i]));
    return __uint_as_float(u);
}

// Least j >= 0 with room * 2^j >= top (both finite, room >= 2^-120).
__device__ __forceinline__ int doublings(float top, float room)
{
    if (top <= room) return 0;
    const uint32_t a = __float_as_uint(top), b = __float_as_uint(room);
    return (int)(a >> 23) - (int)(b >> 23) + ((a & 0x7fffffu) > (b & 0x7fffffu) ? 1 : 0);
}

struct AppendArgs {
    Kv8View w;
    const void* src[2];  // k, v
    long long ld[2];
    int vec[2];
};

// One CTA per (sequence, page of it that rows fall into, head, k or v).
template <typename T>
__global__ void __launch_bounds__(kAppendThreads) k_kv8_append(const AppendArgs a)
{
    __shared__ float red[kAppendThreads / 32];
    pdl_wait();
    const Kv8View& w = a.w;
    const int h = blockIdx.y, kv = blockIdx.z;
    const int span = (w.max_rows + w.P - 2) / w.P + 1;  // pages that max_rows rows can touch
    const int b = blockIdx.x / span;
    const Kv8Seq s = kv8_seq(w, b);
    const int first = max(s.len - s.n, 0), skip = max(s.n - s.len, 0);  // rows before position 0 are skipped
    const int at = (first >> w.lgP) + (int)(blockIdx.x % span);
    const int lo = max(at << w.lgP, first), hi = min((at + 1) << w.lgP, s.len);
    if (hi <= lo) return;
    const int unit = kv8_unit(w, s, at, h);
    if (unit < 0) return;
    const T* src = static_cast<const T*>(a.src[kv]) + (s.row0 + skip + (lo - first)) * a.ld[kv] + (long long)h * w.hd;
    int8_t* page = (kv ? w.v : w.k) + (size_t)unit * w.P * w.hd;
    float* scale = (kv ? w.vs : w.ks) + unit;
    const int q4 = w.hd >> 2, groups = (hi - lo) * q4, had = lo - (at << w.lgP);

    float m = 0.0f;
    bool bad = false;
    for (int g = threadIdx.x; g < groups; g += kAppendThreads) {
        float x[4];
        load4<T>(src + (long long)(g / q4) * a.ld[kv] + (g % q4) * 4, a.vec[kv], x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bad |= !(fabsf(x[i]) <= 3.402823466e38f);
            m = fmaxf(m, fabsf(x[i]));
        }
    }
    const float old = had ? *scale : 0.0f;
    m = block_absmax(m, bad, red);  // also: everybody has read the old scale
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
        for (int g = threadIdx.x; g < had * q4; g += kAppendThreads) {
            char4 c = reinterpret_cast<char4*>(page)[g];
            c.x = (signed char)__float2int_rn(c.x * f);
            c.y = (signed char)__float2int_rn(c.y * f);
            c.z = (signed char)__float2int_rn(c.z * f);
            c.w = (signed char)__float2int_rn(c.w * f);
            reinterpret_cast<char4*>(page)[g] = c;
        }
    }
    const float inv = sc == sc ? __fdiv_rn(1.0f, sc) : 0.0f;
    char4* dst = reinterpret_cast<char4*>(page + (size_t)had * w.hd);
    for (int g = threadIdx.x; g < groups; g += kAppendThreads) {
        float x[4];
        load4<T>(src + (long long)(g / q4) * a.ld[kv] + (g % q4) * 4, a.vec[kv], x);
        int c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = sc == sc ? min(max(__float2int_rn(__fmul_rn(x[i], inv)), -127), 127) : 0;
        dst[g] = make_char4((signed char)c[0], (signed char)c[1], (signed char)c[2], (signed char)c[3]);
    }
    if (threadIdx.x == 0) *scale = sc;
}

// ------------------------------------------------------------------- read --

constexpr int kReadThreads = 256;

struct ReadArgs {
    Kv8View w;
    void* dst[2];
    long long ld[2];
    int vec[2];
};

// Grid: (row chunk of sequence b) x sequences x {k, v}; a thread takes four
// elements of a head of a row.
template <typename T>
__global__ void __launch_bounds__(kReadThreads) k_kv8_read(const ReadArgs a)
{
    pdl_wait();
    const Kv8View& w = a.w;
    const int b = blockIdx.y, kv = blockIdx.z;
    const Kv8Seq s = kv8_seq(w, b);
    const int q4 = w.hd >> 2, per_row = q4 * w.KV;
    for (long long g = blockIdx.x * (long long)kReadThreads + threadIdx.x; g < (long long)s.n * per_row;
         g += (long long)gridDim.x * kReadThreads) {
        const int i = (int)(g / per_row), e = (int)(g % per_row), h = e / q4;
        const int pos = s.len - s.n + i;
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const int unit = pos >= 0 ? kv8_unit(w, s, pos >> w.lgP, h) : -1;
        if (unit >= 0) {
            const size_t off = ((size_t)unit * w.P + (pos & (w.P - 1))) * w.hd + (e % q4) * 4;
            const char4 c = *reinterpret_cast<const char4*>((kv ? w.v : w.k) + off);
            const float sc = (kv ? w.vs : w.ks)[unit];
            x[0] = c.x * sc, x[1] = c.y * sc, x[2] = c.z * sc, x[3] = c.w * sc;
        }
        store4<T>(static_cast<T*>(a.dst[kv]) + (s.row0 + i) * a.ld[kv] + e * 4, a.vec[kv], x);
    }
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
    if ((rc = kv8_check_rows(k, ldk, need)) || (rc = kv8_check_rows(v, ldv, need))) return rc;
    AppendArgs a{};
    a.w = kv8_view(pool, tables, batch, layer);
    const int bytes = type == QUANTR_TYPE_F32 ? 4 : 2;
    a.src[0] = k, a.src[1] = v, a.ld[0] = ldk, a.ld[1] = ldv;
    a.vec[0] = aligned4(k, ldk, bytes), a.vec[1] = aligned4(v, ldv, bytes);
    const long long span = ((long long)batch->max_rows + pool->page_tokens - 2) / pool->page_tokens + 1;
    if (span * batch->B > 0x7fffffffll || pool->n_kv_heads > 65535) return QUANTR_ERR_TOO_LARGE;
    LaunchCfg c;
    c.stream = (cudaStream_t)stream;
    return kv8_done(with_type(type, [&](auto* t) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
        return launch_ex(k_kv8_append<T>, dim3((unsigned)(span * batch->B), pool->n_kv_heads, 2), kAppendThreads, 0, c, a);
    }));
}

int quantr_kv8_read_dev(void* k, long long ldk, void* v, long long ldv, uint32_t type, const quantr_kv8_pool* pool,
                        const quantr_kv8_tables* tables, const quantr_kv8_batch* batch, int layer, void* stream)
{
    int rc = kv8_check_call(pool, tables, batch, layer, type);
    if (rc || batch->B == 0 || batch->max_rows == 0) return rc;
    const long long need = (long long)pool->n_kv_heads * pool->head_dim;
    if ((rc = kv8_check_rows(k, ldk, need)) || (rc = kv8_check_rows(v, ldv, need))) return rc;
    if (batch->B > 65535) return QUANTR_ERR_TOO_LARGE;
    ReadArgs a{};
    a.w = kv8_view(pool, tables, batch, layer);
    const int bytes = type == QUANTR_TYPE_F32 ? 4 : 2;
    a.dst[0] = k, a.dst[1] = v, a.ld[0] = ldk, a.ld[1] = ldv;
    a.vec[0] = aligned4(k, ldk, bytes), a.vec[1] = aligned4(v, ldv, bytes);
    const long long chunks = ((long long)batch->max_rows * (need / 4) + kReadThreads - 1) / kReadThreads;
    LaunchCfg c;
    c.stream = (cudaStream_t)stream;
    return kv8_done(with_type(type, [&](auto* t) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
        return launch_ex(k_kv8_read<T>, dim3((unsigned)std::min(chunks, 4096ll), batch->B, 2), kReadThreads, 0, c, a);
    }));
}

} // extern "C"
