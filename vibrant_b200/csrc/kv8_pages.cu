// kv8_pages.cu -- the pages of the 8-bit KV cache: growing, forking, emptying
// and compacting sequences, without a host read.
//
// A page is free exactly when refs[page] == 0, and free pages are taken lowest
// number first; there is no list that could disagree with the references.
// Choosing pages is one CTA's work (kPlanThreads threads, each over a
// contiguous run of the references: count, one scan over the threads, then the
// numbers in order), so results do not depend on timing; the pool's
// references are a few hundred KB at most, and this costs a few microseconds.
// Moving pages is a grid's work over (page, layer, K or V) pieces, bound by
// bytes: the planner leaves the (from, to) list and its length in the
// workspace and the mover reads them there.  Measured: 60 part-filled pages of
// 64 tokens, 36 layers and 2 heads copied for forks 29 us (4.9 TB/s of reads and
// writes), a pool of 24 sequences packed 44 us (4.0 TB/s, of which the planner
// is some 10 us).
#include <cstdint>

#include "../../include/vkq.h"
#include "kq_device.cuh"
#include "kv8.cuh"
#include "vkq_internal.h"

namespace vkq {

static __device__ int g_kv8_pages_status;

__device__ __forceinline__ void pages_bad() { atomicExch(&g_kv8_pages_status, VKQ_ERR_INVALID_ARGUMENT); }

constexpr int kPlanThreads = 1024;
constexpr int kMoveThreads = 256;

// Workspace, in int32: the number of listed moves, a mark per row (zero
// between calls), then lists of a row's or a page's entries: the moves, the
// free pages found, the lengths of the rows forked.
struct PagesWs {
    int *count, *mark, *from, *to, *found, *len;
};
static int64_t pages_list(int64_t rows, int64_t pages) { return ((rows > pages ? rows : pages) + 3) / 4 * 4; }
static PagesWs pages_ws(void *ws, int64_t rows, int64_t pages) {
    int *w = static_cast<int *>(ws) + 4;
    const int64_t n = pages_list(rows, pages);
    return PagesWs{w - 4, w, w + n, w + 2 * n, w + 3 * n, w + 4 * n};
}
size_t kv8_pages_workspace(const vkq_kv8_cache &c, const vkq_kv8_seqs &q) {
    return (size_t)(4 + 5 * pages_list(q.rows, c.num_pages)) * sizeof(int);
}

struct PagesParams {
    PagesWs ws;
    int *table, *lens, *refs, *done;
    const int *slots, *other;  // add (extend) or src (fork)
    int64_t rows, max_pages, num_pages, n;
    int page;
};

// Exclusive sum over the CTA's threads in order; total: over all of them.
template <typename T>
__device__ T block_scan(T v, T &total) {
    __shared__ T sums[kPlanThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        T s = sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const T y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        sums[lane] = s;
    }
    __syncthreads();
    const T r = x - v + (warp ? sums[warp - 1] : 0);
    total = sums[kPlanThreads / 32 - 1];
    __syncthreads();
    return r;
}

// Lists the lowest free pages, up to `want` of them, in p.ws.found; returns how
// many pages are free.  All threads take part.
__device__ int find_free(const PagesParams &p, int want) {
    const int64_t per = ((p.num_pages + kPlanThreads - 1) / kPlanThreads + 3) / 4 * 4;
    const int64_t a = min((int64_t)threadIdx.x * per, p.num_pages), b = min(a + per, p.num_pages);
    int mine = 0;
    for (int64_t i = a; i < b; i++) mine += p.refs[i] == 0;
    int total, at = block_scan(mine, total);
    if (at < want)
        for (int64_t i = a; i < b && at < want; i++)
            if (p.refs[i] == 0) p.ws.found[at++] = (int)i;
    __syncthreads();
    return total;
}

// Marks the listed rows so that the first mention of a row wins: returns
// whether entry i holds its row.  Entries of other rows give false.
__device__ void mark_rows(const PagesParams &p) {
    for (int64_t i = threadIdx.x; i < p.n; i += kPlanThreads) {
        const int r = p.slots[i];
        if (r >= 0 && r < p.rows) atomicMax(&p.ws.mark[r], (int)(p.n - i));
    }
    __syncthreads();
}
__device__ bool holds_row(const PagesParams &p, int64_t i) {
    const int r = p.slots[i];
    return r >= 0 && r < p.rows && p.ws.mark[r] == (int)(p.n - i);
}
__device__ void clear_marks(const PagesParams &p) {
    __syncthreads();
    for (int64_t i = threadIdx.x; i < p.n; i += kPlanThreads) {
        const int r = p.slots[i];
        if (r >= 0 && r < p.rows) p.ws.mark[r] = 0;
    }
}
__device__ __forceinline__ bool good_len(const PagesParams &p, int len) {
    return len >= 0 && len <= p.max_pages * p.page;
}

__global__ void __launch_bounds__(kPlanThreads) extend_kernel(const PagesParams p) {
    pdl_wait();
    pdl_launch_dependents();
    mark_rows(p);
    // the pages wanted, in all (capped: more than the pool cannot be had)
    __shared__ unsigned long long wanted;
    if (threadIdx.x == 0) wanted = 0;
    __syncthreads();
    auto need = [&](int64_t i, int &len, int &grown, bool &ok) -> int64_t {
        ok = holds_row(p, i);
        if (!ok) return 0;
        len = p.lens[p.slots[i]];
        const int add = p.other[i];
        const int64_t to = (int64_t)len + add;
        ok = add >= 0 && good_len(p, len) && to <= p.max_pages * p.page;
        if (!ok) return 0;
        grown = (int)to;
        return (to + p.page - 1) / p.page - ((int64_t)len + p.page - 1) / p.page;
    };
    for (int64_t i = threadIdx.x; i < p.n; i += kPlanThreads) {
        int len, grown;
        bool ok;
        const int64_t k = need(i, len, grown, ok);
        if (!ok) pages_bad();
        if (k) atomicAdd(&wanted, (unsigned long long)k);
    }
    __syncthreads();
    const int want = (int)min((unsigned long long)p.num_pages, wanted);
    const int have = want ? find_free(p, want) : 0;
    int64_t before = 0;
    for (int64_t i0 = 0; i0 < p.n; i0 += kPlanThreads) {
        const int64_t i = i0 + threadIdx.x;
        int len = 0, grown = 0;
        bool ok = false;
        const int64_t k = i < p.n ? need(i, len, grown, ok) : 0;
        int64_t total;  // a row may grow by 2^26 pages, a thousand of them by more than 2^31
        const int64_t at = before + block_scan(k, total);
        before += total;
        ok = ok && (k == 0 || at + k <= have);
        if (ok) {
            int *row = p.table + (int64_t)p.slots[i] * p.max_pages + (len + p.page - 1) / p.page;
            for (int64_t x = 0; x < k; x++) {
                const int id = p.ws.found[at + x];
                row[x] = id;
                p.refs[id] = 1;
            }
            p.lens[p.slots[i]] = grown;
        }
        if (i < p.n && p.done) p.done[i] = ok;
        __syncthreads();
    }
    clear_marks(p);
}

__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const PagesParams p) {
    pdl_wait();
    pdl_launch_dependents();
    mark_rows(p);
    // p.slots: dst.  A pair is good if dst is empty and src another row of a
    // good length.  part: it needs a page of its own.
    auto good = [&](int64_t i, int &len) {
        if (!holds_row(p, i)) return false;
        const int s = p.other[i], d = p.slots[i];
        if (s < 0 || s >= p.rows || s == d || p.lens[d] != 0) return false;
        len = p.lens[s];
        return good_len(p, len);
    };
    __shared__ int wanted;
    if (threadIdx.x == 0) wanted = 0;
    __syncthreads();
    for (int64_t i = threadIdx.x; i < p.n; i += kPlanThreads) {
        int len = 0;
        const bool ok = good(i, len);
        if (!ok) pages_bad();
        if (ok && len % p.page) atomicAdd(&wanted, 1);
    }
    __syncthreads();
    const int want = (int)min((int64_t)wanted, p.num_pages);
    const int have = want ? find_free(p, want) : 0;
    // ws.from[i], ws.to[i]: the part-filled page and its copy, -1 for none;
    // ws.found past the pages taken is not read again
    int64_t before = 0;
    for (int64_t i0 = 0; i0 < p.n; i0 += kPlanThreads) {
        const int64_t i = i0 + threadIdx.x;
        int len = 0;
        bool ok = i < p.n && good(i, len);
        const int k = ok && len % p.page ? 1 : 0;
        int total;
        const int64_t at = before + block_scan(k, total);
        before += total;
        ok = ok && (k == 0 || at + k <= have);
        if (i < p.n) {
            int f = -1, t = -1;
            if (ok && k) {
                f = p.table[(int64_t)p.other[i] * p.max_pages + len / p.page];
                t = p.ws.found[at];
                p.refs[t] = 1;
            }
            p.ws.from[i] = f;
            p.ws.len[i] = len;  // as it is now: a later pair's src may be an earlier one's dst
            p.ws.to[i] = ok ? t : -2;  // -2: not forked
            if (p.done) p.done[i] = ok;
        }
    }
    clear_marks(p);
}

// One CTA a pair: the row's whole pages are shared, the copy's number entered.
__global__ void __launch_bounds__(kMoveThreads) fork_rows_kernel(const PagesParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t i = blockIdx.x;
    const int t = p.ws.to[i];
    if (t == -2) return;
    const int s = p.other[i], d = p.slots[i];
    const int len = p.ws.len[i], full = len / p.page;
    const int *from = p.table + (int64_t)s * p.max_pages;
    int *to = p.table + (int64_t)d * p.max_pages;
    for (int x = threadIdx.x; x < full; x += kMoveThreads) {
        const int id = from[x];
        to[x] = id;
        if (id >= 0 && id < p.num_pages) atomicAdd(&p.refs[id], 1);
        else pages_bad();
    }
    if (threadIdx.x == 0) {
        if (t >= 0) to[full] = t;
        p.lens[d] = len;
    }
}

// One CTA a row.
__global__ void __launch_bounds__(kMoveThreads) free_kernel(const PagesParams p) {
    __shared__ int len;
    pdl_wait();
    pdl_launch_dependents();
    const int64_t i = blockIdx.x;
    const int r = p.slots[i];
    bool ok = r >= 0 && r < p.rows;
    for (int64_t x = threadIdx.x; ok && x < i; x += kMoveThreads)
        if (p.slots[x] == r) ok = false;  // listed before
    ok = __syncthreads_and(ok);
    if (threadIdx.x == 0) {
        len = ok ? p.lens[r] : 0;
        if (!ok || !good_len(p, len)) pages_bad(), len = 0, ok = false;
        if (ok) p.lens[r] = 0;
        if (p.done) p.done[i] = ok;
    }
    __syncthreads();
    const int pages = (len + p.page - 1) / p.page;
    int *row = p.table + (int64_t)(len ? r : 0) * p.max_pages;
    for (int x = threadIdx.x; x < pages; x += kMoveThreads) {
        const int id = row[x];
        row[x] = -1;
        if (id < 0 || id >= p.num_pages || atomicSub(&p.refs[id], 1) <= 0) {
            if (id >= 0 && id < p.num_pages) atomicAdd(&p.refs[id], 1);  // it had none: keep it free
            pages_bad();
        }
    }
}

// ws.from, ws.to: the moves; ws.found[page]: where a page goes (itself if it stays).
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const PagesParams p, int *used) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t per = ((p.num_pages + kPlanThreads - 1) / kPlanThreads + 3) / 4 * 4;
    const int64_t a = min((int64_t)threadIdx.x * per, p.num_pages), b = min(a + per, p.num_pages);
    int mine = 0, total;
    for (int64_t i = a; i < b; i++) mine += p.refs[i] > 0;
    block_scan(mine, total);
    const int u = total;
    int holes = 0, moves = 0;
    for (int64_t i = a; i < b; i++) {
        const bool in_use = p.refs[i] > 0;
        holes += !in_use && i < u;
        moves += in_use && i >= u;
    }
    int all;
    int h = block_scan(holes, all);
    int m = block_scan(moves, all);
    for (int64_t i = a; i < b; i++) {
        const bool in_use = p.refs[i] > 0;
        if (!in_use && i < u) p.ws.to[h++] = (int)i;
        if (in_use && i >= u) p.ws.from[m++] = (int)i;
    }
    __syncthreads();
    for (int64_t i = threadIdx.x; i < p.num_pages; i += kPlanThreads) p.ws.found[i] = (int)i;
    __syncthreads();
    for (int x = threadIdx.x; x < all; x += kPlanThreads) {
        const int f = p.ws.from[x], t = p.ws.to[x];
        p.ws.found[f] = t;
        p.refs[t] = p.refs[f];
        p.refs[f] = 0;
    }
    if (threadIdx.x == 0) {
        *p.ws.count = all;
        if (used) *used = u;
    }
}

__global__ void __launch_bounds__(kMoveThreads) rename_kernel(const PagesParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t all = p.rows * p.max_pages;
    for (int64_t i = (int64_t)blockIdx.x * kMoveThreads + threadIdx.x; i < all; i += (int64_t)gridDim.x * kMoveThreads) {
        const int id = p.table[i];
        if (id >= 0 && id < p.num_pages && p.ws.found[id] != id) p.table[i] = p.ws.found[id];
    }
}

struct MoveParams {
    uint8_t *k, *v;
    float *ks, *vs;
    int64_t num_pages, layers, n;
    int64_t page_codes, page_scales;  // of one page and layer: bytes, floats
    const int *from, *to, *count;     // count NULL: n moves
    bool holes;                       // entries with to < 0 are no moves
};

// A CTA takes pieces (move, layer, K or V) of whole pages: a page's codes are
// contiguous in a layer, 16 bytes a thread and pass, four in flight.
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const MoveParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t moves = p.count ? *p.count : p.n;
    const int64_t pieces = moves * p.layers * 2;
    for (int64_t x = blockIdx.x; x < pieces; x += gridDim.x) {
        const int64_t m = x / (2 * p.layers);
        const int rest = (int)(x - m * 2 * p.layers);
        const int64_t f = p.from[m], t = p.to[m];
        if (p.holes && t < 0) continue;
        if (f < 0 || f >= p.num_pages || t < 0 || t >= p.num_pages) {
            if (threadIdx.x == 0) pages_bad();
            continue;
        }
        const int64_t layer = rest >> 1;
        uint8_t *codes = ((rest & 1) ? p.v : p.k) + layer * p.num_pages * p.page_codes;
        float *scales = ((rest & 1) ? p.vs : p.ks) + layer * p.num_pages * p.page_scales;
        const uint4 *src = reinterpret_cast<const uint4 *>(codes + f * p.page_codes);
        uint4 *dst = reinterpret_cast<uint4 *>(codes + t * p.page_codes);
        const int n16 = (int)(p.page_codes / 16);
        for (int i = threadIdx.x; i < n16; i += 4 * kMoveThreads) {
            uint4 r[4];
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (i + u * kMoveThreads < n16) r[u] = src[i + u * kMoveThreads];
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (i + u * kMoveThreads < n16) dst[i + u * kMoveThreads] = r[u];
        }
        for (int i = threadIdx.x; i < p.page_scales; i += kMoveThreads)
            scales[t * p.page_scales + i] = scales[f * p.page_scales + i];
    }
}

static cudaError_t launch(const void *fn, int64_t blocks, int threads, void **args, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelExC(&cfg, fn, args);
}

static PagesParams pages_params(const vkq_kv8_cache &c, const vkq_kv8_seqs &q, const int *slots, const int *other,
                                int64_t n, int *done, void *ws) {
    PagesParams p{};
    p.ws = pages_ws(ws, q.rows, c.num_pages);
    p.table = q.table, p.lens = q.lens, p.refs = q.refs, p.done = done;
    p.slots = slots, p.other = other;
    p.rows = q.rows, p.max_pages = q.max_pages, p.num_pages = c.num_pages, p.n = n;
    p.page = c.page_size;
    return p;
}

// The mover's grid: a CTA a piece of `moves` at most, and no more than the eight
// of 256 threads that an SM holds, to hide a page's latency behind another's.
static cudaError_t launch_move(const vkq_kv8_cache &c, const int *from, const int *to, const int *count, int64_t moves,
                               bool holes, cudaStream_t s, int device) {
    MoveParams p{};
    p.k = static_cast<uint8_t *>(c.k), p.v = static_cast<uint8_t *>(c.v);
    p.ks = c.k_scale, p.vs = c.v_scale;
    p.num_pages = c.num_pages, p.layers = c.layers, p.n = moves;
    p.page_codes = (int64_t)c.kv_heads * c.page_size * c.head_dim;
    p.page_scales = (int64_t)c.kv_heads * (c.page_size / kKv8Block);
    p.from = from, p.to = to, p.count = count, p.holes = holes;
    int64_t blocks = moves * c.layers * 2;
    const int64_t cap = 8 * (int64_t)device_sm_count(device);
    if (blocks > cap) blocks = cap;
    void *args[] = {&p};
    return launch((const void *)move_kernel, blocks, kMoveThreads, args, s);
}

cudaError_t kv8_extend(const vkq_kv8_cache &c, const vkq_kv8_seqs &q, const int *slots, const int *add, int64_t n,
                       int *done, void *ws, cudaStream_t s) {
    PagesParams p = pages_params(c, q, slots, add, n, done, ws);
    void *args[] = {&p};
    return launch((const void *)extend_kernel, 1, kPlanThreads, args, s);
}

cudaError_t kv8_fork(const vkq_kv8_cache &c, const vkq_kv8_seqs &q, const int *src, const int *dst, int64_t n, int *done,
                     void *ws, cudaStream_t s, int device) {
    PagesParams p = pages_params(c, q, dst, src, n, done, ws);
    void *args[] = {&p};
    cudaError_t e = launch((const void *)fork_plan_kernel, 1, kPlanThreads, args, s);
    if (e == cudaSuccess) e = launch((const void *)fork_rows_kernel, n, kMoveThreads, args, s);
    if (e == cudaSuccess) e = launch_move(c, p.ws.from, p.ws.to, nullptr, n, true, s, device);
    return e;
}

cudaError_t kv8_free(const vkq_kv8_cache &c, const vkq_kv8_seqs &q, const int *slots, int64_t n, int *done, void *ws,
                     cudaStream_t s) {
    PagesParams p = pages_params(c, q, slots, nullptr, n, done, ws);
    void *args[] = {&p};
    return launch((const void *)free_kernel, n, kMoveThreads, args, s);
}

cudaError_t kv8_compact(const vkq_kv8_cache &c, const vkq_kv8_seqs &q, int *used, void *ws, cudaStream_t s, int device) {
    PagesParams p = pages_params(c, q, nullptr, nullptr, 0, nullptr, ws);
    void *args[] = {&p, &used};
    cudaError_t e = launch((const void *)compact_plan_kernel, 1, kPlanThreads, args, s);
    if (e == cudaSuccess) {
        int64_t blocks = (q.rows * q.max_pages + kMoveThreads - 1) / kMoveThreads;
        const int64_t cap = 8 * (int64_t)device_sm_count(device);
        if (blocks > cap) blocks = cap;
        e = launch((const void *)rename_kernel, blocks, kMoveThreads, args, s);
    }
    if (e == cudaSuccess) e = launch_move(c, p.ws.from, p.ws.to, p.ws.count, (c.num_pages + 1) / 2, false, s, device);
    return e;
}

cudaError_t kv8_copy_pages(const vkq_kv8_cache &c, const int *src, const int *dst, int64_t n, cudaStream_t s, int device) {
    return launch_move(c, src, dst, nullptr, n, false, s, device);
}

int *kv8_pages_status_word() { return status_word(g_kv8_pages_status); }

}  // namespace vkq
