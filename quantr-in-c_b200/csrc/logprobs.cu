// logprobs.cu -- log probabilities of given tokens, entropy and the k largest
// alternatives of rows of logits (public contract: include/quantr_cuda.h).
#include "kv8.cuh"

#include <cmath>

namespace qr {
namespace {

constexpr int kLpThreads = 512;

struct LpArgs {
    const void* x;
    long long ldl;
    int rows, V, k;
    float inv_t;
    const int* token;
    float* logprob;
    float* entropy;
    float* lse;
    int* top_id;
    float* top_lp;
};

// Order of alternatives: larger logits first, then lower ids.  0 is below all
// (-inf and NaN are not alternatives).
__device__ __forceinline__ unsigned long long lp_key(float x, int id)
{
    if (!(x > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(x + 0.0f);  // -0 is 0
    const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (unsigned long long)o << 32 | (uint32_t)~id;
}

// One CTA per row: maximum; sums; then k passes, each for the largest key
// below the last.
template <typename T>
__global__ void __launch_bounds__(kLpThreads) k_logprobs(const LpArgs a)
{
    __shared__ float fr[kLpThreads / 32], gr[kLpThreads / 32];
    __shared__ unsigned long long kr[kLpThreads / 32];
    pdl_wait();
    const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const T* x = static_cast<const T*>(a.x) + row * a.ldl;
    float m = -INFINITY;
    bool bad = false;
    for (int v = tid; v < a.V; v += kLpThreads) {
        const float y = to_f<T>(x[v]) * a.inv_t;
        bad |= !(y < INFINITY);
        m = fmaxf(m, y);
    }
    for (int z = 16; z; z >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, z));
    if (lane == 0) fr[warp] = m;
    bad = __syncthreads_or(bad);
    for (int i = 0; i < kLpThreads / 32; ++i) m = fmaxf(m, fr[i]);
    __syncthreads();
    float s = 0.0f, e = 0.0f;
    if (m > -INFINITY && !bad)
        for (int v = tid; v < a.V; v += kLpThreads) {
            const float d = to_f<T>(x[v]) * a.inv_t - m, p = expf(d);
            s += p;
            if (p > 0.0f) e = fmaf(p, d, e);
        }
    for (int z = 16; z; z >>= 1) s += __shfl_xor_sync(~0u, s, z), e += __shfl_xor_sync(~0u, e, z);
    if (lane == 0) fr[warp] = s, gr[warp] = e;
    __syncthreads();
    s = e = 0.0f;
    for (int i = 0; i < kLpThreads / 32; ++i) s += fr[i], e += gr[i];
    float lse = m + logf(s), ent = logf(s) - e / s;
    if (m == -INFINITY) lse = -INFINITY, ent = 0.0f;
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
    unsigned long long last = ~0ull;
    for (int j = 0; j < a.k; ++j) {
        unsigned long long best = 0;
        for (int v = tid; v < a.V; v += kLpThreads) {
            const unsigned long long key = lp_key(to_f<T>(x[v]), v);
            if (key < last && key > best) best = key;
        }
        for (int z = 16; z; z >>= 1) best = max(best, __shfl_xor_sync(~0u, best, z));
        if (lane == 0) kr[warp] = best;
        __syncthreads();
        for (int i = 0; i < kLpThreads / 32; ++i) best = max(best, kr[i]);
        __syncthreads();
        last = best;
        if (tid == 0) {
            const int id = best ? (int)~(uint32_t)best : -1;
            if (a.top_id) a.top_id[(long long)row * a.k + j] = id;
            if (a.top_lp) a.top_lp[(long long)row * a.k + j] = id < 0 ? (bad ? NAN : -INFINITY)
                                                                      : to_f<T>(x[id]) * a.inv_t - lse;
        }
        if (!best) last = 0;
    }
}

} // namespace
} // namespace qr

extern "C" {

using namespace qr;

size_t quantr_logprobs_workspace_bytes(int rows, int vocab, int k)
{
    (void)rows, (void)vocab, (void)k;
    return 256;
}

int quantr_logprobs_dev(const void* x, long long ldl, uint32_t type, int rows, int vocab, float temperature,
                        const int* token, float* logprob, float* entropy, float* lse, int k, int* top_id,
                        float* top_logprob, void* workspace, size_t workspace_bytes, void* stream)
{
    if (!kv8_float_type(type)) return QUANTR_ERR_UNSUPPORTED_TYPE;
    if (rows < 0 || vocab <= 0 || k < 0 || ldl < vocab || !(temperature > 0.0f) || !std::isfinite(temperature) ||
        !std::isfinite(1.0f / temperature))
        return QUANTR_ERR_BAD_ARG;
    if (k > 64) return QUANTR_ERR_TOO_LARGE;
    if (rows == 0) return QUANTR_OK;
    if (!x || (logprob && !token)) return QUANTR_ERR_BAD_ARG;
    if (!workspace || ((uintptr_t)workspace & 255) ||
        workspace_bytes < quantr_logprobs_workspace_bytes(rows, vocab, k))
        return QUANTR_ERR_WORKSPACE;
    LpArgs a{x,     ldl,     rows, vocab,  k, (float)(1.0 / (double)temperature), token, logprob, entropy, lse, top_id,
             top_logprob};
    LaunchCfg c;
    c.stream = (cudaStream_t)stream;
    cudaError_t e = with_type(type, [&](auto* t) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
        return launch_ex(k_logprobs<T>, dim3(rows), kLpThreads, 0, c, a);
    });
    return kv8_done(e);
}

} // extern "C"
