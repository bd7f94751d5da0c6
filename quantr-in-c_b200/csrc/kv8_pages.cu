// kv8_pages.cu -- page operators of the 8-bit paged KV cache: select (fork,
// free, reorder), extend, compact, copy (public contract:
// include/quantr_cuda.h).
#include "kv8.cuh"

#include <algorithm>

namespace qr {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;

// Exclusive prefix sum over the CTA's threads; `total` to all.
__device__ int block_scan(int v, int* total, int* red /* 33 ints */)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(~0u, x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();  // red may still be read from an earlier scan
    if (lane == 31) red[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int s = lane < (int)blockDim.x / 32 ? red[lane] : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(~0u, s, d);
            if (lane >= d) s += y;
        }
        red[lane] = s;
    }
    __syncthreads();
    *total = red[blockDim.x / 32 - 1];
    return x - v + (warp ? red[warp - 1] : 0);
}

// ----------------------------------------------------------------- select --

struct SelectArgs {
    quantr_kv8_tables to, in;
    const int* from;
    int n_pages, lgP;
    int* err;
};

constexpr int kSelectCtas = 8, kSelectThreads = 1024;

// One cluster: the references are zeroed, the cluster meets, and its warps take
// the slots one by one, counting the pages they copy (integers: their order does
// not matter).  Latency-bound: 3.7 us for 64 slots of 10 to
// 18 pages, 2.2 for 16 of 9.
__global__ void __launch_bounds__(kSelectThreads) __cluster_dims__(kSelectCtas, 1, 1) k_kv8_select(const SelectArgs a)
{
    pdl_wait();
    const int lane = threadIdx.x & 31, P = 1 << a.lgP;
    for (int i = blockIdx.x * kSelectThreads + threadIdx.x; i < a.n_pages; i += kSelectCtas * kSelectThreads)
        a.to.refs[i] = 0;
    cluster_arrive();
    cluster_wait();
    for (int s = (blockIdx.x * kSelectThreads + threadIdx.x) >> 5; s < a.to.slots; s += kSelectCtas * kSelectThreads / 32) {
        int f = a.from[s];
        if (f < -1 || f >= a.in.slots) {
            kv8_fault(a.err);
            f = -1;
        }
        int len = f >= 0 ? a.in.lens[f] : 0;
        if (len < 0 || (long long)len > ((long long)a.in.max_pages << a.lgP)) {
            kv8_fault(a.err);
            len = 0;
        }
        const int used = (int)(((long long)len + P - 1) >> a.lgP);
        const int* in = a.in.table + (size_t)max(f, 0) * a.in.max_pages;
        int* to = a.to.table + (size_t)s * a.to.max_pages;
#pragma unroll 4
        for (int i = lane; i < a.in.max_pages; i += 32) {
            const int page = i < used ? in[i] : -1;
            to[i] = page;
            if (page >= 0 && page < a.n_pages) atomicAdd(a.to.refs + page, 1);
            else if (i < used) kv8_fault(a.err);
        }
        if (lane == 0) a.to.lens[s] = len;
    }
}

// ----------------------------------------------------------- page copying --

// A list of copies, in the workspace of the planning kernels: head[0] = how
// many; pair i copies page src[i] to dst[i].
struct CopyArgs {
    quantr_kv8_pool pool;
    const int* count;
    int n;  // with count null
    const int* src;
    const int* dst;
    int* err;
    // Compaction: the tables' entries follow the map (null: none).
    int* table;
    const int* map;
    size_t entries;
};

constexpr int kAtOnce = 4;                      // 16-byte loads in flight per thread
constexpr int kChunk = kCopyThreads * kAtOnce;  // vectors that a CTA copies at a time (16 KB)

// Work item (copy, chunk of its page): 16 KB of codes, or the page's scales.
// CTAs take the items in turn, so a few large pages fill the GPU as well as
// many small ones.  Memory-bound: 250 pages of 3.1 MB, 1.57 GB read and written,
// in 245 us, 6.4 TB/s.
__global__ void __launch_bounds__(kCopyThreads) k_kv8_copy(const CopyArgs a)
{
    pdl_wait();
    const quantr_kv8_pool& p = a.pool;
    const int n = a.count ? *a.count : a.n;
    const size_t units = (size_t)p.n_layers * p.n_kv_heads, vecs = units * p.page_tokens * p.head_dim / 16;
    const int chunks = (int)((vecs + kChunk - 1) / kChunk), items = 2 * chunks + 1;
    for (long long w = blockIdx.x; w < (long long)n * items; w += gridDim.x) {
        const int i = (int)(w / items), c = (int)(w - (long long)i * items);
        const int src = a.src[i], dst = a.dst[i];
        if (src < 0 || src >= p.n_pages || dst < 0 || dst >= p.n_pages) {
            kv8_fault(a.err);
            continue;
        }
        if (c == 2 * chunks) {
            for (size_t j = threadIdx.x; j < units; j += kCopyThreads) {
                p.k_scale[dst * units + j] = p.k_scale[src * units + j];
                p.v_scale[dst * units + j] = p.v_scale[src * units + j];
            }
            continue;
        }
        int8_t* codes = c < chunks ? p.k : p.v;
        const uint4* s = reinterpret_cast<const uint4*>(codes) + src * vecs;
        uint4* d = reinterpret_cast<uint4*>(codes) + dst * vecs;
        const size_t at = (size_t)(c < chunks ? c : c - chunks) * kChunk + threadIdx.x;
        uint4 v[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
            if (at + j * kCopyThreads < vecs) v[j] = s[at + j * kCopyThreads];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
            if (at + j * kCopyThreads < vecs) d[at + j * kCopyThreads] = v[j];
    }
    if (a.map)
        for (size_t i = (size_t)blockIdx.x * kCopyThreads + threadIdx.x; i < a.entries;
             i += (size_t)gridDim.x * kCopyThreads) {
            const int page = a.table[i];
            if (page >= 0 && page < p.n_pages) a.table[i] = a.map[page];
        }
}

// ----------------------------------------------------------------- extend --

struct PlanArgs {
    quantr_kv8_tables t;
    int n_pages, lgP, B;
    const int* slot;
    const int* n_new;
    int* grown;
    int* count;  // copies; then the lists
    int* src;
    int* dst;
    int* list;  // extend: free pages; compact: the map
    int* n_live;
    int* map;
    int* err;
};

// One CTA, thread i plans sequence i: what it needs, a prefix sum of that, the
// free pages up to the total.  Latency-bound: with its copies (15 pages of 0.7
// MB, 22 MB moved) an extend of 16 sequences takes 7.8 us.
__global__ void __launch_bounds__(kPlanThreads) k_kv8_extend(const PlanArgs a)
{
    __shared__ int red[33], tails[kPlanThreads];
    __shared__ int found_s;
    __shared__ bool failed[kPlanThreads];
    pdl_wait();
    const int i = threadIdx.x, P = 1 << a.lgP;
    int slot = -1, len = 0, n = 0, tail = -1;
    bool ok = false;
    if (i < a.B) {
        slot = a.slot ? a.slot[i] : i;
        n = a.n_new ? a.n_new[i] : 1;
        if (slot < 0 || slot >= a.t.slots || n < 0) {
            kv8_fault(a.err);
        } else {
            len = a.t.lens[slot];
            ok = len >= 0 && (long long)len + n <= ((long long)a.t.max_pages << a.lgP);
            if (!ok) kv8_fault(a.err);
            if (ok && n > 0 && (len & (P - 1))) {
                tail = a.t.table[(size_t)slot * a.t.max_pages + (len >> a.lgP)];
                if (tail < 0 || tail >= a.n_pages) {
                    kv8_fault(a.err);
                    ok = false;
                    tail = -1;
                }
            }
        }
    }
    int* row = a.t.table + (size_t)max(slot, 0) * a.t.max_pages;
    tails[i] = tail;
    __syncthreads();
    // A shared last page is copied unless only this sequence is left on it
    // when its turn comes.
    bool copied = false;
    if (tail >= 0) {
        int earlier = 0;
        for (int j = 0; j < i; ++j) earlier += tails[j] == tail;
        copied = a.t.refs[tail] - earlier > 1;
    }
    const int old_pages = (int)(((long long)len + P - 1) >> a.lgP);
    const int new_pages = ok ? (int)(((long long)len + n + P - 1) >> a.lgP) : old_pages;
    const int need = ok ? (copied ? 1 : 0) + (new_pages - old_pages) : 0;
    int total;
    const int base = block_scan(need, &total, red);
    // The free pages of lowest index, in order, until there are enough.
    int found = 0;
    for (int p0 = 0; p0 < a.n_pages && found < total; p0 += 4 * kPlanThreads) {
        const int page = p0 + 4 * i;
        int is[4], mine = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            is[j] = page + j < a.n_pages && a.t.refs[page + j] == 0;
            mine += is[j];
        }
        int sum;
        int at = found + block_scan(mine, &sum, red);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (is[j]) {
                if (at < total) a.list[at] = page + j;
                ++at;
            }
        found += sum;
    }
    if (i == 0) found_s = found;
    __syncthreads();
    // Out of pages: for this sequence and for every later one that needs one.
    // Who would have kept a shared page as the last of its holders needs one,
    // too, if one of the others got no copy.
    const bool late = ok && need > 0 && base + need > found_s;
    failed[i] = late;
    __syncthreads();
    bool left = false;
    if (ok && tail >= 0 && !copied)
        for (int j = 0; j < i; ++j) left |= tails[j] == tail && failed[j];
    if (late || left) {
        kv8_fault(a.err);
        ok = false;
    }
    copied = copied && ok;
    int copies;
    const int c = block_scan(copied, &copies, red);
    if (i == 0) *a.count = copies;
    if (ok) {
        int at = base;
        if (copied) {
            const int page = a.list[at++];
            a.src[c] = tail;
            a.dst[c] = page;
            row[len >> a.lgP] = page;
            a.t.refs[page] = 1;
            atomicSub(a.t.refs + tail, 1);
        }
        for (int j = old_pages; j < new_pages; ++j) {
            const int page = a.list[at++];
            row[j] = page;
            a.t.refs[page] = 1;
        }
        a.t.lens[slot] = len + n;
    }
    if (a.grown && i < a.B) a.grown[i] = ok;
}

// ---------------------------------------------------------------- compact --

// One CTA: n_live, then the i-th page in use at or past it to the i-th hole
// before it: the fewest pages move, and none is read and written.  With the
// copies, 1.69 GB read and written: 263 us, 6.4 TB/s.
__global__ void __launch_bounds__(kPlanThreads) k_kv8_compact(const PlanArgs a)
{
    __shared__ int red[33];
    pdl_wait();
    int live = 0;
    for (int p0 = 0; p0 < a.n_pages; p0 += 4 * kPlanThreads) {
        const int page = p0 + 4 * threadIdx.x;
        int mine = 0, sum;
#pragma unroll
        for (int j = 0; j < 4; ++j) mine += page + j < a.n_pages && a.t.refs[page + j] > 0;
        block_scan(mine, &sum, red);
        live += sum;
    }
    // Holes and movers counted in one number each time: at most 4096 of either.
    int holes = 0, movers = 0;
    for (int p0 = 0; p0 < a.n_pages; p0 += 4 * kPlanThreads) {
        const int page = p0 + 4 * threadIdx.x;
        bool used[4];
        int mine = 0, sum;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            used[j] = page + j < a.n_pages && a.t.refs[page + j] > 0;
            if (page + j < live && !used[j]) mine += 1;
            if (page + j >= live && used[j]) mine += 1 << 16;
        }
        const int at = block_scan(mine, &sum, red);
        int hole = holes + (at & 0xffff), mover = movers + (at >> 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (page + j < live && !used[j]) a.dst[hole++] = page + j;
            if (page + j >= live && used[j]) a.src[mover++] = page + j;
            if (page + j < a.n_pages) a.list[page + j] = used[j] ? page + j : -1;
        }
        holes += sum & 0xffff;
        movers += sum >> 16;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < movers; i += kPlanThreads) {
        const int src = a.src[i], dst = a.dst[i];
        a.list[src] = dst;
        a.t.refs[dst] = a.t.refs[src];
        a.t.refs[src] = 0;
    }
    __syncthreads();
    if (a.map)
        for (int i = threadIdx.x; i < a.n_pages; i += kPlanThreads) a.map[i] = a.list[i];
    if (threadIdx.x == 0) {
        *a.count = movers;
        if (a.n_live) *a.n_live = live;
    }
}

int lg_tokens(const quantr_kv8_pool* p) { return p->page_tokens == 32 ? 5 : p->page_tokens == 64 ? 6 : 7; }

// CTAs for at most `pages` copies: 32 per SM (several waves: their ends overlap
// better than those of CTAs that stay; 4 per SM measured 7 % slower), fewer where
// there is less to do.
int copy_grid(const quantr_kv8_pool* p, long long pages)
{
    const long long vecs = (long long)p->n_layers * p->n_kv_heads * p->page_tokens * p->head_dim / 16;
    const long long items = std::max(pages, 1ll) * (2 * ((vecs + kChunk - 1) / kChunk) + 1);
    return (int)std::min<long long>(items, 32ll * device_sm_count());
}

// Workspace: count, then src, dst and list of n_pages each.
struct PagesWs {
    int *count, *src, *dst, *list;
};

PagesWs carve(void* ws, int n_pages)
{
    const size_t n = ((size_t)n_pages + 63) & ~size_t(63);
    int* p = static_cast<int*>(ws);
    return {p, p + 64, p + 64 + n, p + 64 + 2 * n};
}

} // namespace
} // namespace qr

extern "C" {

using namespace qr;

int quantr_kv8_select_dev(const quantr_kv8_tables* to, const quantr_kv8_tables* in, const int* from,
                          const quantr_kv8_pool* pool, void* stream)
{
    int rc = kv8_check_pool(pool);
    if (!rc) rc = kv8_check_tables(to);
    if (!rc) rc = kv8_check_tables(in);
    if (rc) return rc;
    if (!from || to->slots != in->slots || to->max_pages != in->max_pages || to->table == in->table ||
        to->lens == in->lens || to->refs == in->refs || !kv8_aligned({from}))
        return QUANTR_ERR_BAD_ARG;
    SelectArgs a{*to, *in, from, pool->n_pages, lg_tokens(pool), device_error_word()};
    LaunchCfg c;
    c.stream = (cudaStream_t)stream;
    return kv8_done(launch_ex(k_kv8_select, dim3(kSelectCtas), kSelectThreads, 0, c, a));
}

size_t quantr_kv8_pages_workspace_bytes(const quantr_kv8_pool* pool, const quantr_kv8_tables* tables)
{
    (void)tables;
    if (!pool || pool->n_pages <= 0) return 0;
    return 256 + 3 * 4 * (((size_t)pool->n_pages + 63) & ~size_t(63));
}

static int pages_check(const quantr_kv8_pool* pool, const quantr_kv8_tables* t, const void* ws, size_t bytes)
{
    int rc = kv8_check_pool(pool);
    if (!rc) rc = kv8_check_tables(t);
    if (rc) return rc;
    if (!ws || ((uintptr_t)ws & 255) || bytes < quantr_kv8_pages_workspace_bytes(pool, t)) return QUANTR_ERR_WORKSPACE;
    return QUANTR_OK;
}

static PlanArgs plan_args(const quantr_kv8_pool* pool, const quantr_kv8_tables* t, void* ws)
{
    PlanArgs a{};
    const PagesWs w = carve(ws, pool->n_pages);
    a.t = *t;
    a.n_pages = pool->n_pages;
    a.lgP = lg_tokens(pool);
    a.count = w.count, a.src = w.src, a.dst = w.dst, a.list = w.list;
    a.err = device_error_word();
    return a;
}

int quantr_kv8_extend_dev(const quantr_kv8_pool* pool, const quantr_kv8_tables* tables, const int* slot,
                          const int* n_new, int B, int* grown, void* workspace, size_t workspace_bytes, void* stream)
{
    int rc = pages_check(pool, tables, workspace, workspace_bytes);
    if (!rc && (B < 0 || (!slot && B > tables->slots) || !kv8_aligned({slot, n_new, grown}))) rc = QUANTR_ERR_BAD_ARG;
    if (!rc && B > kPlanThreads) rc = QUANTR_ERR_TOO_LARGE;
    if (rc || B == 0) return rc;
    PlanArgs a = plan_args(pool, tables, workspace);
    a.B = B, a.slot = slot, a.n_new = n_new, a.grown = grown;
    LaunchCfg c;
    c.stream = (cudaStream_t)stream;
    cudaError_t e = launch_ex(k_kv8_extend, dim3(1), kPlanThreads, 0, c, a);
    CopyArgs k{*pool, a.count, 0, a.src, a.dst, a.err, nullptr, nullptr, 0};
    if (e == cudaSuccess) e = launch_ex(k_kv8_copy, dim3(copy_grid(pool, B)), kCopyThreads, 0, c, k);
    return kv8_done(e);
}

int quantr_kv8_compact_dev(const quantr_kv8_pool* pool, const quantr_kv8_tables* tables, int* map, int* n_live,
                           void* workspace, size_t workspace_bytes, void* stream)
{
    int rc = pages_check(pool, tables, workspace, workspace_bytes);
    if (!rc && !kv8_aligned({map, n_live})) rc = QUANTR_ERR_BAD_ARG;
    if (rc) return rc;
    PlanArgs a = plan_args(pool, tables, workspace);
    a.map = map, a.n_live = n_live;
    LaunchCfg c;
    c.stream = (cudaStream_t)stream;
    cudaError_t e = launch_ex(k_kv8_compact, dim3(1), kPlanThreads, 0, c, a);
    CopyArgs k{*pool, a.count, 0, a.src, a.dst, a.err, tables->table, a.list, (size_t)tables->slots * tables->max_pages};
    if (e == cudaSuccess) e = launch_ex(k_kv8_copy, dim3(copy_grid(pool, pool->n_pages)), kCopyThreads, 0, c, k);
    return kv8_done(e);
}

int quantr_kv8_copy_pages_dev(const quantr_kv8_pool* pool, const int* dst, const int* src, int n, void* stream)
{
    int rc = kv8_check_pool(pool);
    if (!rc && (n < 0 || (n > 0 && (!dst || !src)) || !kv8_aligned({dst, src}))) rc = QUANTR_ERR_BAD_ARG;
    if (rc || n == 0) return rc;
    CopyArgs k{*pool, nullptr, n, src, dst, device_error_word(), nullptr, nullptr, 0};
    LaunchCfg c;
    c.stream = (cudaStream_t)stream;
    return kv8_done(launch_ex(k_kv8_copy, dim3(copy_grid(pool, n)), kCopyThreads, 0, c, k));
}

} // extern "C"
