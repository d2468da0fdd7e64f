// kv8_cache.cu -- writing new tokens into the 8-bit paged KV cache (rotated,
// quantized by blocks of 16 tokens and head) and reading rows back.
//
// Append.  Block (sequence, 16 tokens, KV head) of K or V: with a the largest
// finite magnitude among its new tokens,
//   s_new = least 2^e with a <= m 2^e,  s = max(s_old, s_new) if the block
//   holds older tokens, else s_new;  code = round(x / s)
// and, where s grew, the older codes become round(code * s_old / s).  Scales
// are powers of two: x / s is then exact, so a code is rounded once, and a
// block filled token by token has each code rounded again at most when the
// scale doubles, which bounds what its roundings add up to by one step of the
// last scale (with free scales, 15 appends could add 15 half steps).  The cost
// is up to one bit of the int8 code's range; e4m3 loses nothing.
//
// One warp takes one block of K or V: the 16 rows sit in its registers
// (D / 32 values of each row a lane), the maximum is one butterfly, and no
// other warp touches the block, so there are no atomics and the result does
// not depend on the order of anything.  Bytes bound a prompt, latency a decode
// step; q's rotation rides in the same launch (warps past the blocks'), which
// saves a launch a layer.
#include <cstdint>

#include "../../include/vkq.h"
#include "act.cuh"
#include "kq_device.cuh"
#include "kv8.cuh"
#include "vkq_internal.h"

namespace vkq {

static __device__ int g_kv8_status;

__device__ __forceinline__ void kv8_bad() { atomicExch(&g_kv8_status, VKQ_ERR_INVALID_ARGUMENT); }

constexpr int kAppThreads = 128;
constexpr int kAppWarps = kAppThreads / 32;

struct AppendParams {
    Kv8Pool pool;
    Kv8Batch batch;
    const void *k, *v, *q;
    void *q_out;
    int64_t kt, vt, qt, qot;  // token strides, in elements
    const float *cos_t, *sin_t;
    int64_t max_seq;
    int heads, rot;
    int max_blocks;       // blocks that one sequence's new tokens can touch
    int64_t block_items;  // warps of blocks: batch * max_blocks * kv_heads * 2
    int64_t items;        // and of q: tokens * ceil(heads / kAppHeads)
    bool half, vec_kv, vec_q;
};
constexpr int kAppHeads = 4;  // heads of q that a warp rotates

// The lane's N = D / 32 values of one row, rotated at position ps (table row):
// interleaved pairs lie in the lane; a half pair's partner is loaded as well.
// Any rot: values past it are as they are.
template <typename T, int D>
__device__ __forceinline__ void load_turned(const T *row, float (&x)[D / 32], int lane, bool vec, bool rotate,
                                            const float *cos_t, const float *sin_t, int64_t ps, int rot, bool half) {
    constexpr int N = D / 32;
    const int d0 = lane * N, h = rot / 2;
    load_act<T, N>(row + d0, x, vec);
    if (!rotate) return;
    const float *ct = cos_t + ps * h, *st = sin_t + ps * h;
    if (!half) {
#pragma unroll
        for (int i = 0; i < N; i += 2)
            if (d0 + i < rot) turn(x[i], x[i + 1], ct[(d0 + i) / 2], st[(d0 + i) / 2]);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int d = d0 + i;
        if (d < h) {
            float b = to_f32<T>(row[d + h]);
            turn(x[i], b, ct[d], st[d]);
        } else if (d < rot) {
            float a = to_f32<T>(row[d - h]);
            turn(a, x[i], ct[d - h], st[d - h]);
        }
    }
}

template <typename T, int D>
__device__ void append_block(const AppendParams &p, int64_t item, int lane) {
    constexpr int N = D / 32;
    const bool is_v = item & 1;
    int64_t r = item >> 1;
    const int kvh = p.pool.kv_heads;
    const int h = (int)(r % kvh);
    r /= kvh;
    const int j = (int)(r % p.max_blocks);
    const int64_t b = r / p.max_blocks;
    const Kv8Seq s = kv8_seq(p.batch, p.pool.page, b);
    const bool rotate = p.cos_t != nullptr;
    if (!s.ok || s.n > s.len || (rotate && s.len > p.max_seq)) {
        if (lane == 0 && j == 0) kv8_bad();
        return;
    }
    const int start = s.len - s.n;
    const int blk = start / kKv8Block + j;
    const int pos0 = blk * kKv8Block;
    if (s.n == 0 || pos0 >= s.len) return;
    const int lo = max(start - pos0, 0), hi = min(s.len - pos0, kKv8Block);  // the block's new rows
    const int id = kv8_page(p.pool, s, pos0 / p.pool.page);
    if (id < 0) {
        if (lane == 0) kv8_bad();
        return;
    }
    const int in_page = pos0 % p.pool.page;
    const int64_t ph = (int64_t)id * kvh + h;
    float *scale = (is_v ? p.pool.vs : p.pool.ks) + ph * (p.pool.page / kKv8Block) + in_page / kKv8Block;
    uint8_t *codes = (is_v ? p.pool.v : p.pool.k) + (ph * p.pool.page + in_page) * D + lane * N;
    const T *src = static_cast<const T *>(is_v ? p.v : p.k) + (int64_t)(s.first + pos0 - start) * (is_v ? p.vt : p.kt) +
                   h * D;
    const int64_t stride = is_v ? p.vt : p.kt;
    const float s_old = lo > 0 ? *scale : 0.f;
    float x[kKv8Block][N];
    float a = 0.f;
#pragma unroll
    for (int t = 0; t < kKv8Block; t++) {
        if (t >= lo && t < hi) {
            load_turned<T, D>(src + t * stride, x[t], lane, p.vec_kv, rotate && !is_v, p.cos_t, p.sin_t, pos0 + t, p.rot,
                              p.half);
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float m = fabsf(x[t][i]);
                if (m <= 3.402823466e38f) a = fmaxf(a, m);  // finite
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) x[t][i] = 0.f;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
    const float sc = fmaxf(s_old, kv8_scale(a, p.pool.e4m3));
    if (lo > 0 && sc > s_old) {
        const float ratio = __fdiv_rn(s_old, sc);
        for (int t = 0; t < lo; t++) {
            uint8_t *c = codes + t * D;
            uint32_t w = N == 4 ? *reinterpret_cast<uint32_t *>(c) : *reinterpret_cast<uint16_t *>(c), o = 0;
#pragma unroll
            for (int i = 0; i < N; i++)
                o |= kv8_encode(kv8_decode((w >> (8 * i)) & 0xFFu, p.pool.e4m3) * ratio, p.pool.e4m3) << (8 * i);
            if (N == 4) *reinterpret_cast<uint32_t *>(c) = o;
            else *reinterpret_cast<uint16_t *>(c) = (uint16_t)o;
        }
    }
    const float inv = __fdiv_rn(1.f, sc);
#pragma unroll
    for (int t = 0; t < kKv8Block; t++) {
        if (t < lo || t >= hi) continue;
        uint32_t o = 0;
#pragma unroll
        for (int i = 0; i < N; i++) o |= kv8_encode(x[t][i] * inv, p.pool.e4m3) << (8 * i);
        if (N == 4) *reinterpret_cast<uint32_t *>(codes + t * D) = o;
        else *reinterpret_cast<uint16_t *>(codes + t * D) = (uint16_t)o;
    }
    if (lane == 0) *scale = sc;
}

// The sequence of token t: the last b with cu[b] <= t (empty sequences skipped).
__device__ __forceinline__ int64_t seq_of_token(const Kv8Batch &b, int64_t t) {
    if (!b.cu) return t;
    int64_t lo = 0, hi = b.batch;  // cu[lo] <= t < cu[hi] where the offsets are in order
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) / 2;
        if (b.cu[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <typename T, int D>
__device__ void append_q(const AppendParams &p, int64_t item, int lane) {
    constexpr int N = D / 32;
    const int groups = (p.heads + kAppHeads - 1) / kAppHeads;
    const int64_t t = item / groups;
    const int h0 = (int)(item - t * groups) * kAppHeads;
    const int64_t b = seq_of_token(p.batch, t);
    if (b >= p.batch.batch) return;
    const Kv8Seq s = kv8_seq(p.batch, p.pool.page, b);
    if (!s.ok || s.n > s.len || s.len > p.max_seq || t < s.first || t >= s.first + s.n) return;
    const int64_t ps = s.len - s.n + (t - s.first);
    const T *q = static_cast<const T *>(p.q) + t * p.qt;
    T *o = static_cast<T *>(p.q_out) + t * p.qot;
    float x[kAppHeads][N];
#pragma unroll
    for (int u = 0; u < kAppHeads; u++)
        if (h0 + u < p.heads)
            load_turned<T, D>(q + (h0 + u) * D, x[u], lane, p.vec_q, true, p.cos_t, p.sin_t, ps, p.rot, p.half);
    __syncwarp();  // q_out may be q: a lane has read its partner before any lane writes
#pragma unroll
    for (int u = 0; u < kAppHeads; u++)
        if (h0 + u < p.heads) store_act<T, N>(o + (h0 + u) * D + lane * N, x[u], p.vec_q);
}

template <typename T, int D>
__global__ void __launch_bounds__(kAppThreads) append_kernel(const AppendParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t item = (int64_t)blockIdx.x * kAppWarps + (threadIdx.x >> 5);
    if (item < p.block_items) append_block<T, D>(p, item, lane);
    else if (item < p.items) append_q<T, D>(p, item - p.block_items, lane);
}

// ---- reading rows back ------------------------------------------------------
struct ReadParams {
    Kv8Pool pool;
    Kv8Batch batch;
    const int *seq, *pos;
    int64_t items;  // n * kv_heads * D / 4
    void *k_out, *v_out;
};

// Four values a thread: bytes bound it, and consecutive threads write 16 (8)
// consecutive bytes each.
template <typename T>
__global__ void __launch_bounds__(256) read_kernel(const ReadParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int quads = p.pool.D / 4, kvh = p.pool.kv_heads;
    for (int64_t it = (int64_t)blockIdx.x * 256 + threadIdx.x; it < p.items; it += (int64_t)gridDim.x * 256) {
        const int64_t row = it / ((int64_t)quads * kvh);
        const int rest = (int)(it - row * quads * kvh);
        const int h = rest / quads, d = (rest - h * quads) * 4;
        const int64_t b = p.seq[row];
        const int ps = p.pos[row];
        int id = -1;
        if (b >= 0 && b < p.batch.batch) {
            const Kv8Seq s = kv8_seq(p.batch, p.pool.page, b);
            if (s.ok && ps >= 0 && ps < s.len) id = kv8_page(p.pool, s, ps / p.pool.page);
        }
        float kx[4], vx[4];
        if (id < 0) {
            if (rest == 0) kv8_bad();
            kx[0] = kx[1] = kx[2] = kx[3] = vx[0] = vx[1] = vx[2] = vx[3] = __int_as_float(0x7fc00000);
        } else {
            const int at = ps % p.pool.page;
            const int64_t ph = (int64_t)id * kvh + h;
            const int64_t e = (ph * p.pool.page + at) * p.pool.D + d, se = ph * (p.pool.page / kKv8Block) + at / kKv8Block;
            const uint32_t kw = *reinterpret_cast<const uint32_t *>(p.pool.k + e);
            const uint32_t vw = *reinterpret_cast<const uint32_t *>(p.pool.v + e);
            const float ks = p.pool.ks[se], vs = p.pool.vs[se];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                kx[i] = kv8_decode((kw >> (8 * i)) & 0xFFu, p.pool.e4m3) * ks;
                vx[i] = kv8_decode((vw >> (8 * i)) & 0xFFu, p.pool.e4m3) * vs;
            }
        }
        if (p.k_out) store_act<T, 4>(static_cast<T *>(p.k_out) + it * 4, kx, true);
        if (p.v_out) store_act<T, 4>(static_cast<T *>(p.v_out) + it * 4, vx, true);
    }
}

static cudaError_t launch(const void *fn, int64_t blocks, int threads, void *params, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    void *args[] = {params};
    return cudaLaunchKernelExC(&cfg, fn, args);
}

template <typename T>
static const void *append_fn(int D) {
    return D == 64 ? (const void *)append_kernel<T, 64> : (const void *)append_kernel<T, 128>;
}

int64_t kv8_append_warps(const vkq_kv8_cache &c, const vkq_kv8_batch &b, int64_t heads, bool q) {
    const int64_t max_blocks = (b.max_tokens + kKv8Block - 2) / kKv8Block + 1;
    return b.batch * max_blocks * c.kv_heads * 2 + (q ? b.tokens * ((heads + kAppHeads - 1) / kAppHeads) : 0);
}

cudaError_t kv8_append(const vkq_kv8_cache &c, int64_t layer, const vkq_kv8_batch &b, const Kv8AppendArgs &a,
                       cudaStream_t s) {
    AppendParams p{};
    p.pool = kv8_pool(c, layer);
    p.batch = kv8_batch(b);
    p.k = a.k, p.v = a.v, p.q = a.q, p.q_out = a.q_out;
    p.kt = a.k_token, p.vt = a.v_token, p.qt = a.q_token, p.qot = a.q_out_token;
    p.cos_t = a.cos_t, p.sin_t = a.sin_t, p.max_seq = a.max_seq;
    p.heads = (int)a.heads, p.rot = (int)a.rot_dim, p.half = a.layout == VKQ_ROPE_HALF;
    p.max_blocks = (int)((b.max_tokens + kKv8Block - 2) / kKv8Block + 1);
    p.block_items = b.batch * p.max_blocks * c.kv_heads * 2;
    p.items = kv8_append_warps(c, b, a.heads, a.q != nullptr);
    // a lane's D / 32 values as one vector
    const int size = act_bytes(a.dtype);
    const uintptr_t lane = (uintptr_t)(c.head_dim / 32 * size) - 1;
    p.vec_kv = (((uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)(a.k_token * size) | (uintptr_t)(a.v_token * size)) & lane) == 0;
    p.vec_q = (((uintptr_t)a.q | (uintptr_t)a.q_out | (uintptr_t)(a.q_token * size) | (uintptr_t)(a.q_out_token * size)) &
               lane) == 0;
    const void *fn = a.dtype == VKQ_F32   ? append_fn<float>(c.head_dim)
                     : a.dtype == VKQ_F16 ? append_fn<__half>(c.head_dim)
                                          : append_fn<__nv_bfloat16>(c.head_dim);
    return launch(fn, (p.items + kAppWarps - 1) / kAppWarps, kAppThreads, &p, s);
}

cudaError_t kv8_read(const vkq_kv8_cache &c, int64_t layer, const vkq_kv8_batch &b, const int *seq, const int *pos,
                     int64_t n, int dtype, void *k_out, void *v_out, cudaStream_t s, int device) {
    ReadParams p{};
    p.pool = kv8_pool(c, layer);
    p.batch = kv8_batch(b);
    p.seq = seq, p.pos = pos, p.k_out = k_out, p.v_out = v_out;
    p.items = n * c.kv_heads * (c.head_dim / 4);
    int64_t blocks = (p.items + 255) / 256;
    const int64_t cap = 64 * (int64_t)device_sm_count(device);
    if (blocks > cap) blocks = cap;
    const void *fn = dtype == VKQ_F32   ? (const void *)read_kernel<float>
                     : dtype == VKQ_F16 ? (const void *)read_kernel<__half>
                                        : (const void *)read_kernel<__nv_bfloat16>;
    return launch(fn, blocks, 256, &p, s);
}

int kv8_read_status() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_kv8_status, sizeof(int)) != cudaSuccess) return -1;
    cudaMemcpyToSymbol(g_kv8_status, &zero, sizeof(int));
    return v;
}

}  // namespace vkq
