// kv8.cuh -- what the kernels of the 8-bit paged KV cache share: views of the
// public descriptors, their checks, and typed element access.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <initializer_list>

#include "device_common.cuh"
#include "kernels.cuh"
#include "launch_util.cuh"

namespace qr {

constexpr uint32_t T_F16 = QUANTR_TYPE_F16, T_BF16 = QUANTR_TYPE_BF16;

inline bool kv8_float_type(uint32_t t) { return t == QUANTR_TYPE_F32 || t == T_F16 || t == T_BF16; }

// Whether all addresses (null ones too) are multiples of an element's size: an
// access at any other is a fault on the device.
inline bool kv8_aligned(std::initializer_list<const void*> ps, size_t bytes = 4)
{
    for (const void* p : ps)
        if ((uintptr_t)p % bytes) return false;
    return true;
}

inline int kv8_check_pool(const quantr_kv8_pool* p)
{
    if (!p || !p->k || !p->v || !p->k_scale || !p->v_scale) return QUANTR_ERR_BAD_ARG;
    if (!kv8_aligned({p->k, p->v}, 16) || !kv8_aligned({p->k_scale, p->v_scale})) return QUANTR_ERR_BAD_ARG;
    if (p->n_pages <= 0 || p->n_layers <= 0 || p->n_kv_heads <= 0) return QUANTR_ERR_BAD_ARG;
    if (p->page_tokens != 32 && p->page_tokens != 64 && p->page_tokens != 128) return QUANTR_ERR_BAD_ARG;
    if (p->head_dim <= 0 || p->head_dim % 16) return QUANTR_ERR_BAD_ARG;
    if (p->head_dim > 128) return QUANTR_ERR_TOO_LARGE;
    if ((double)p->n_pages * p->n_layers * p->n_kv_heads >= 2147483648.0) return QUANTR_ERR_TOO_LARGE;
    return QUANTR_OK;
}

inline int kv8_check_tables(const quantr_kv8_tables* t)
{
    if (!t || !t->table || !t->lens || !t->refs || t->slots <= 0 || t->max_pages <= 0) return QUANTR_ERR_BAD_ARG;
    return kv8_aligned({t->table, t->lens, t->refs}) ? QUANTR_OK : QUANTR_ERR_BAD_ARG;
}

// A batch of no sequences or no rows is allowed (the calls do nothing).
inline int kv8_check_batch(const quantr_kv8_batch* b)
{
    if (!b || b->B < 0 || b->max_rows < 0 || !kv8_aligned({b->slot, b->start})) return QUANTR_ERR_BAD_ARG;
    // Row numbers are 32-bit, those that `start` gives already.
    return b->start || (long long)b->B * b->max_rows <= 0x7fffffffll ? QUANTR_OK : QUANTR_ERR_TOO_LARGE;
}

inline size_t kv8_type_bytes(uint32_t type) { return type == QUANTR_TYPE_F32 ? 4 : 2; }

inline int kv8_check_rows(const void* p, long long ld, long long need, uint32_t type)
{
    return p && ld >= need && kv8_aligned({p}, kv8_type_bytes(type)) ? QUANTR_OK : QUANTR_ERR_BAD_ARG;
}

inline int kv8_check_call(const quantr_kv8_pool* pool, const quantr_kv8_tables* tables, const quantr_kv8_batch* batch, int layer,
               uint32_t type)
{
    int rc = kv8_check_pool(pool);
    if (!rc) rc = kv8_check_tables(tables);
    if (!rc) rc = kv8_check_batch(batch);
    if (!rc && (layer < 0 || layer >= pool->n_layers)) rc = QUANTR_ERR_BAD_ARG;
    if (!rc && !kv8_float_type(type)) rc = QUANTR_ERR_UNSUPPORTED_TYPE;
    return rc;
}

inline int kv8_done(cudaError_t e)
{
    if (e != cudaSuccess) cudaGetLastError();
    return status_code(e);
}

// The cache as kernels see it: one layer's scales and codes are reached by the
// unit (page*n_layers + layer)*n_kv_heads + head, a 31-bit number; byte offsets
// are 64-bit.
struct Kv8View {
    int8_t* k;
    int8_t* v;
    float* ks;
    float* vs;
    int n_pages, L, KV, P, lgP, hd;
    const int* table;
    const int* lens;
    int slots, max_pages;
    const int* slot;
    const int* start;
    int B, max_rows;
    int layer;
    int* err;
};

inline Kv8View kv8_view(const quantr_kv8_pool* p, const quantr_kv8_tables* t, const quantr_kv8_batch* b, int layer)
{
    Kv8View w{};
    w.k = p->k;
    w.v = p->v;
    w.ks = p->k_scale;
    w.vs = p->v_scale;
    w.n_pages = p->n_pages;
    w.L = p->n_layers;
    w.KV = p->n_kv_heads;
    w.P = p->page_tokens;
    w.lgP = p->page_tokens == 32 ? 5 : p->page_tokens == 64 ? 6 : 7;
    w.hd = p->head_dim;
    w.table = t->table;
    w.lens = t->lens;
    w.slots = t->slots;
    w.max_pages = t->max_pages;
    w.slot = b->slot;
    w.start = b->start;
    w.B = b->B;
    w.max_rows = b->max_rows;
    w.layer = layer;
    w.err = device_error_word();
    return w;
}

__device__ __forceinline__ void kv8_fault(int* err)
{
    if (err) atomicCAS(err, (int)DEV_OK, (int)DEV_ERR_PAGES);
}

// One sequence of the batch: its table row (null: no such slot), its length (0
// where it is below), its rows row0 .. row0+n-1, the first of which stands at
// position len - n.
struct Kv8Seq {
    const int* pages;
    int len, n, row0;
};

__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8View& w, int b)
{
    Kv8Seq s;
    const int slot = w.slot ? w.slot[b] : b;
    if (w.start) {
        s.row0 = w.start[b];
        s.n = min(max(w.start[b + 1] - s.row0, 0), w.max_rows);
    } else {
        s.row0 = b * w.max_rows;
        s.n = w.max_rows;
    }
    if (slot < 0 || slot >= w.slots) {
        s.pages = nullptr;
        s.len = 0;
        kv8_fault(w.err);
        return s;
    }
    s.pages = w.table + (size_t)slot * w.max_pages;
    s.len = w.lens[slot];
    if (s.len < 0 || (long long)s.len > (long long)w.max_pages * w.P) kv8_fault(w.err);
    s.len = max(s.len, 0);
    return s;
}

// Unit of head h of page `at` of the sequence (its at-th page), or -1 where
// there is none.
__device__ __forceinline__ int kv8_unit(const Kv8View& w, const Kv8Seq& s, int at, int h)
{
    if (!s.pages || at < 0 || at >= w.max_pages) return -1;
    const int page = s.pages[at];
    if (page < 0 || page >= w.n_pages) {
        kv8_fault(w.err);
        return -1;
    }
    return (page * w.L + w.layer) * w.KV + h;
}

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Four consecutive elements; `vec`: the address is aligned to all four.
template <typename T>
__device__ __forceinline__ void load4(const T* p, bool vec, float (&x)[4])
{
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(p);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
        } else {
            const uint2 a = *reinterpret_cast<const uint2*>(p);
            const T* t = reinterpret_cast<const T*>(&a);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = to_f<T>(t[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = to_f<T>(p[i]);
    }
}

// Whether rows of `ld` elements of `bytes` each begin at multiples of `to`.
inline bool aligned(const void* p, long long ld, int bytes, int to) { return (uintptr_t)p % to == 0 && ld * bytes % to == 0; }

// Calls f with a null T* of the element type.
template <typename F>
cudaError_t with_type(uint32_t type, F&& f)
{
    if (type == QUANTR_TYPE_F32) return f((const float*)nullptr);
    if (type == T_F16) return f((const __half*)nullptr);
    return f((const __nv_bfloat16*)nullptr);
}

} // namespace qr
