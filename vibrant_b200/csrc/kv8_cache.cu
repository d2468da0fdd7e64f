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
// A CTA takes K or V of one head of a block, or one after another of all heads:
// four rows a warp (D / 32 values of a row a lane), the maximum over the warps
// through shared memory.  No other CTA touches its items, so there are no
// atomics and the result does not depend on the order of anything.  Latency
// bounds a decode step (48 sequences: 10 us with the read-back), the
// instructions a value a prompt (20,133 tokens in bfloat16, 8 KV heads and q's
// 40: 145 us); q's rotation rides in the same launch (CTAs past the blocks', a
// few tokens each), which saves a launch a layer.
#include <cstdint>

#include "../../include/vkq.h"
#include "act.cuh"
#include "kq_device.cuh"
#include "kv8.cuh"
#include "rotary.cuh"
#include "vkq_internal.h"

namespace vkq {

static __device__ int g_kv8_status;

__device__ __forceinline__ void kv8_bad() { atomicExch(&g_kv8_status, VKQ_ERR_INVALID_ARGUMENT); }

constexpr int kAppThreads = 128;
constexpr int kAppWarps = kAppThreads / 32;

constexpr int kAppRows = kKv8Block / kAppWarps;  // rows of a block that a warp takes

struct AppendParams {
    Kv8Pool pool;
    Kv8Batch batch;
    const void *k, *v, *q;
    void *q_out;
    int64_t kt, vt, qt, qot;  // token strides, in elements
    const float *cos_t, *sin_t;
    int64_t max_seq;
    int heads, rot;
    uint32_t max_blocks;   // blocks that one sequence's new tokens can touch
    int items;             // (K or V, head) of a block that a CTA takes, and the CTAs that this makes
    uint32_t groups, block_ctas;  // block_ctas = batch * max_blocks * groups
    uint32_t magic_groups, magic_blocks, magic_page;  // of groups, max_blocks, page / 16 (kv8_div)
    int q_tokens, q_items; // tokens of a CTA of q's, items of a token
    bool half, vec_kv, vec_t, vec_q;  // a lane's values as one vector: k and v, the tables; q by 16-byte pieces
};
constexpr int kAppMaxTokens = 8;

// How a lane's N = D / 32 values of a head turn: interleaved pairs lie in the
// lane, a half pair's partners in another lane's row part (loaded as well).
// `vec`: the lane's values have one role, so partners and table entries are
// vectors; else each value is looked at by itself.
struct LaneTurn {
    int d0, h, rot;    // the lane's first dimension; rot / 2; rot
    bool rotate, half, vec;
};
template <int N>
__device__ __forceinline__ LaneTurn lane_turn(const AppendParams &p, int lane, bool rotate) {
    return LaneTurn{lane * N, p.rot / 2, p.rot, rotate, p.half, p.rot % (2 * N) == 0 && p.vec_t};
}
// The table entries of the lane's values at position ps (vec only).
template <int N>
__device__ __forceinline__ void load_entries(const AppendParams &p, const LaneTurn &l, int64_t ps, float (&c)[N],
                                             float (&s)[N]) {
    if (!l.rotate || !l.vec || l.d0 >= l.rot) return;
    const int64_t row = ps * l.h;
    if (l.half) {
        const int64_t e = row + (l.d0 < l.h ? l.d0 : l.d0 - l.h);
        load_act<float, N>(p.cos_t + e, c, true);
        load_act<float, N>(p.sin_t + e, s, true);
        if (l.d0 < l.h)
#pragma unroll
            for (int i = 0; i < N; i++) s[i] = -s[i];
    } else {
        float a[N / 2], b[N / 2];
        if constexpr (N == 4) {
            const float2 x = *reinterpret_cast<const float2 *>(p.cos_t + row + l.d0 / 2);
            const float2 y = *reinterpret_cast<const float2 *>(p.sin_t + row + l.d0 / 2);
            a[0] = x.x, a[1] = x.y, b[0] = y.x, b[1] = y.y;
        } else {
            a[0] = p.cos_t[row + l.d0 / 2], b[0] = p.sin_t[row + l.d0 / 2];
        }
#pragma unroll
        for (int i = 0; i < N / 2; i++) c[i] = a[i], s[i] = b[i];
    }
}
// N elements as they are in memory, in words.
template <typename T, int N>
struct Raw {
    static constexpr int W = N * (int)sizeof(T) / 4;  // 1, 2 or 4
    uint32_t w[W];
    __device__ __forceinline__ void load(const T *p, bool vec) {
        if (vec) {
            if constexpr (W == 4) {
                const uint4 x = *reinterpret_cast<const uint4 *>(p);
                w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
            } else if constexpr (W == 2) {
                const uint2 x = *reinterpret_cast<const uint2 *>(p);
                w[0] = x.x, w[1] = x.y;
            } else {
                w[0] = *reinterpret_cast<const uint32_t *>(p);
            }
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < W; i++) w[i] = *reinterpret_cast<const uint32_t *>(p + i);
        } else {
            const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
            for (int i = 0; i < W; i++) w[i] = (uint32_t)h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
        }
    }
    __device__ __forceinline__ void get(float (&x)[N]) const {
        const T *v = reinterpret_cast<const T *>(w);
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = to_f32<T>(v[i]);
    }
};
template <typename T, int N>
__device__ __forceinline__ void turn_lane(const AppendParams &p, const T *row, const LaneTurn &l, int64_t ps,
                                          const float (&c)[N], const float (&s)[N], float (&x)[N], float (&y)[N]) {
    if (!l.rotate || l.d0 >= l.rot) return;
    if (l.vec) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (l.half) {  // s of the first half comes negated: x c - y s is x c + y (-s)
                x[i] = __fadd_rn(__fmul_rn(x[i], c[i]), __fmul_rn(y[i], s[i]));
            } else if (i % 2 == 0) {
                turn(x[i], x[i + 1], c[i / 2], s[i / 2]);
            }
        }
        return;
    }
    const float *ct = p.cos_t + ps * l.h, *st = p.sin_t + ps * l.h;
    for (int i = 0; i < N; i++) {
        const int d = l.d0 + i;
        if (d >= l.rot) break;
        if (!l.half) {
            if (i % 2 == 0) turn(x[i], x[i + 1], ct[d / 2], st[d / 2]);
        } else if (d < l.h) {
            float b = to_f32<T>(row[d + l.h]);
            turn(x[i], b, ct[d], st[d]);
        } else {
            float a = to_f32<T>(row[d - l.h]);
            turn(a, x[i], ct[d - l.h], st[d - l.h]);
        }
    }
}

template <typename T, int D>
__device__ void append_block(const AppendParams &p, uint32_t cta) {
    constexpr int N = D / 32;
    __shared__ float amax[2][kAppWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int kvh = p.pool.kv_heads;
    // the CTA's block, and which of its items (the K heads, then the V heads)
    const uint32_t r = kv8_div(cta, p.groups, p.magic_groups);
    const int i0 = (int)(cta - r * p.groups) * p.items, i1 = min(i0 + p.items, 2 * kvh);
    const uint32_t seq = kv8_div(r, p.max_blocks, p.magic_blocks);
    const int j = (int)(r - seq * p.max_blocks);
    const Kv8Seq s = kv8_seq(p.batch, p.pool.page, seq);
    const bool rotate = p.cos_t != nullptr;
    if (!s.ok || s.n > s.len || (rotate && s.len > p.max_seq)) {
        if (threadIdx.x == 0 && j == 0) kv8_bad();
        return;
    }
    const int start = s.len - s.n;
    const int pos0 = (start / kKv8Block + j) * kKv8Block;
    if (s.n == 0 || pos0 >= s.len) return;
    const int lo = max(start - pos0, 0), hi = min(s.len - pos0, kKv8Block);  // the block's new rows
    const int64_t row0 = (int64_t)(s.first + pos0 - start);
    const LaneTurn lt_k = lane_turn<N>(p, lane, rotate), lt_v = lane_turn<N>(p, lane, false);
    const bool pairs = lt_k.rotate && lt_k.vec && lt_k.half && lt_k.d0 < lt_k.rot;
    const int partner = lt_k.d0 < lt_k.h ? lt_k.d0 + lt_k.h : lt_k.d0 - lt_k.h;
    // the rows of an item; the next item's are under way while one is worked on
    Raw<T, N> xr[kAppRows], yr[kAppRows];
    auto load = [&](int it) {
        const bool is_v = it >= kvh;
        const int64_t stride = is_v ? p.vt : p.kt;
        const T *src = static_cast<const T *>(is_v ? p.v : p.k) + row0 * stride + (is_v ? it - kvh : it) * D;
#pragma unroll
        for (int i = 0; i < kAppRows; i++) {
            const int t = warp + i * kAppWarps;
            if (t < lo || t >= hi) continue;
            xr[i].load(src + t * stride + lane * N, p.vec_kv);
            if (pairs && !is_v) yr[i].load(src + t * stride + partner, p.vec_kv);
        }
    };
    load(i0);
    float c[kAppRows][N], sn[kAppRows][N];  // all K heads turn alike
#pragma unroll
    for (int i = 0; i < kAppRows; i++) {
        const int t = warp + i * kAppWarps;
        if (t >= lo && t < hi && i0 < kvh) load_entries<N>(p, lt_k, pos0 + t, c[i], sn[i]);
    }
    const uint32_t per_page = (uint32_t)(p.pool.page / kKv8Block), blk = (uint32_t)(pos0 / kKv8Block);
    const uint32_t lp = kv8_div(blk, per_page, p.magic_page);
    const int id = kv8_page(p.pool, s, (int)lp);
    if (id < 0) {
        if (threadIdx.x == 0) kv8_bad();
        return;
    }
    const int64_t at0 = (int64_t)id * kvh * per_page + (blk - lp * per_page);
#pragma unroll 1
    for (int it = i0; it < i1; it++) {
        const bool is_v = it >= kvh;
        const int h = is_v ? it - kvh : it;
        const int64_t at = at0 + (int64_t)h * per_page, stride = is_v ? p.vt : p.kt;
        float *scale = (is_v ? p.pool.vs : p.pool.ks) + at;
        uint8_t *codes = (is_v ? p.pool.v : p.pool.k) + at * (kKv8Block * D) + lane * N;
        const T *src = static_cast<const T *>(is_v ? p.v : p.k) + row0 * stride + h * D;
        const float s_old = lo > 0 ? *scale : 0.f;
        float x[kAppRows][N];
        float a = 0.f, z = 0.f;  // z: 0, or NaN after a value that is no number or infinite
#pragma unroll
        for (int i = 0; i < kAppRows; i++) {
            const int t = warp + i * kAppWarps;
            if (t < lo || t >= hi) continue;
            float y[N];
            xr[i].get(x[i]);
            yr[i].get(y);
            turn_lane<T, N>(p, src + t * stride, is_v ? lt_v : lt_k, pos0 + t, c[i], sn[i], x[i], y);
#pragma unroll
            for (int u = 0; u < N; u++) {
                a = fmaxf(a, fabsf(x[i][u]));
                z = fmaf(x[i][u], 0.f, z);
            }
        }
        if (it + 1 < i1) load(it + 1);
        const bool odd = __syncthreads_or(!(z == 0.f));
        if (odd) {  // the largest of the finite ones
            a = 0.f;
#pragma unroll
            for (int i = 0; i < kAppRows; i++) {
                const int t = warp + i * kAppWarps;
#pragma unroll
                for (int u = 0; u < N; u++)
                    if (t >= lo && t < hi && fabsf(x[i][u]) <= 3.402823466e38f) a = fmaxf(a, fabsf(x[i][u]));
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
        if (lane == 0) amax[it & 1][warp] = a;
        __syncthreads();  // every thread has read the old scale, too
#pragma unroll
        for (int w = 0; w < kAppWarps; w++) a = fmaxf(a, amax[it & 1][w]);
        const float sc = fmaxf(s_old, kv8_scale(a, p.pool.e4m3));
        const bool grew = lo > 0 && sc > s_old;
        const uint32_t bits = __float_as_uint(sc);  // of a power of two: the inverse is one subtraction
        const float inv = (bits & 0x7fffffu) == 0 ? __uint_as_float(0x7f000000u - bits) : __fdiv_rn(1.f, sc);
        const float ratio = grew ? __fdiv_rn(s_old, sc) : 1.f;
        const bool saturates = odd || sc >= kKv8MaxScale;
#pragma unroll
        for (int i = 0; i < kAppRows; i++) {
            const int t = warp + i * kAppWarps;
            if (t >= hi || (t < lo && !grew)) continue;
            uint8_t *out = codes + t * D;
            uint32_t o = 0;
            if (t < lo) {
                const uint32_t w = N == 4 ? *reinterpret_cast<uint32_t *>(out) : *reinterpret_cast<uint16_t *>(out);
#pragma unroll
                for (int u = 0; u < N; u++)
                    o |= kv8_encode(kv8_decode((w >> (8 * u)) & 0xFFu, p.pool.e4m3) * ratio, p.pool.e4m3) << (8 * u);
            } else if (saturates) {
#pragma unroll
                for (int u = 0; u < N; u++) o |= kv8_encode(x[i][u] * inv, p.pool.e4m3) << (8 * u);
            } else {
                o = kv8_encode4(x[i][0] * inv, x[i][1] * inv, N == 4 ? x[i][N - 2] * inv : 0.f,
                                N == 4 ? x[i][N - 1] * inv : 0.f, p.pool.e4m3);
            }
            if (N == 4) *reinterpret_cast<uint32_t *>(out) = o;
            else *reinterpret_cast<uint16_t *>(out) = (uint16_t)o;
        }
        if (threadIdx.x == 0) *scale = sc;
    }
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

// q_tokens tokens of q: their positions first, then the items of all of them.
template <typename T, int D>
__device__ void append_q(const AppendParams &p, uint32_t cta) {
    __shared__ int pos[kAppMaxTokens];
    const int64_t t0 = (int64_t)cta * p.q_tokens;
    if ((int)threadIdx.x < p.q_tokens) {
        const int64_t t = t0 + threadIdx.x, b = t < p.batch.tokens ? seq_of_token(p.batch, t) : p.batch.batch;
        int at = -1;
        if (b < p.batch.batch) {
            const Kv8Seq s = kv8_seq(p.batch, p.pool.page, b);
            if (s.ok && s.n <= s.len && s.len <= p.max_seq && t >= s.first && t < s.first + s.n)
                at = s.len - s.n + (int)(t - s.first);
        }
        pos[threadIdx.x] = at;
    }
    __syncthreads();
    const int groups = (p.heads + kRotHeads - 1) / kRotHeads;
    for (int x = threadIdx.x; x < p.q_tokens * p.q_items; x += kAppThreads) {
        const int i = x / p.q_items, rest = x - i * p.q_items;
        if (pos[i] < 0) continue;
        const T *q = static_cast<const T *>(p.q) + (t0 + i) * p.qt;
        T *o = static_cast<T *>(p.q_out) + (t0 + i) * p.qot;
        if (p.vec_q) {
            const int pieces = p.q_items / groups, g = rest / pieces, j = rest - g * pieces, h0 = g * kRotHeads;
            auto row = [&]() -> int64_t { return pos[i]; };
            if (p.half)
                rotary_item<T, true>(q + h0 * D, D, o + h0 * D, D, p.heads - h0, j, D, p.rot, p.cos_t, p.sin_t, false, row);
            else
                rotary_item<T, false>(q + h0 * D, D, o + h0 * D, D, p.heads - h0, j, D, p.rot, p.cos_t, p.sin_t, false, row);
        } else {
            const int per = D - p.rot / 2, h = rest / per;
            rotary_one<T>(q + h * D, o + h * D, rest - h * per, p.rot, p.half, p.cos_t, p.sin_t, false, pos[i]);
        }
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kAppThreads, 6) append_kernel(const AppendParams p) {
    pdl_wait();
    pdl_launch_dependents();
    if (blockIdx.x < p.block_ctas) append_block<T, D>(p, blockIdx.x);
    else append_q<T, D>(p, blockIdx.x - p.block_ctas);
}

// ---- reading rows back ------------------------------------------------------
struct ReadParams {
    Kv8Pool pool;
    Kv8Batch batch;
    const int *seq, *pos;
    int64_t n;
    int rows;  // of a CTA
    void *k_out, *v_out;
};
constexpr int kReadThreads = 256, kReadRows = 8;

// A CTA takes eight rows (one, where there are few): one thread a row finds its page, then every thread
// reads the same four values of each row.  Bytes bound it; consecutive threads
// write 16 (8) consecutive bytes each.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(kReadThreads) read_kernel(const ReadParams p) {
    __shared__ int64_t row_at[kReadRows], scale_at[kReadRows];  // of KV head 0
    pdl_wait();
    pdl_launch_dependents();
    const int64_t r0 = (int64_t)blockIdx.x * p.rows;
    const int D = p.pool.D, page = p.pool.page;
    if ((int)threadIdx.x < p.rows) {
        int64_t at = -1, sc = 0;
        const int64_t r = r0 + threadIdx.x;
        if (r < p.n) {
            const int64_t b = p.seq[r];
            const int ps = p.pos[r];
            if (b >= 0 && b < p.batch.batch) {
                const Kv8Seq s = kv8_seq(p.batch, page, b);
                if (s.ok && ps >= 0 && ps < s.len) {
                    const int id = kv8_page(p.pool, s, ps / page), in = ps % page;
                    if (id >= 0) {
                        at = ((int64_t)id * p.pool.kv_heads * page + in) * D;
                        sc = (int64_t)id * p.pool.kv_heads * (page / kKv8Block) + in / kKv8Block;
                    }
                }
            }
            if (at < 0) kv8_bad();
        }
        row_at[threadIdx.x] = at;
        scale_at[threadIdx.x] = sc;
    }
    __syncthreads();
    const int quads = D / 4, width = p.pool.kv_heads * quads, rows = (int)min((int64_t)p.rows, p.n - r0);
    for (int x = threadIdx.x; x < width; x += kReadThreads) {
        const int h = x / quads, d = (x - h * quads) * 4;
        uint32_t kw[kReadRows], vw[kReadRows];
        float ks[kReadRows], vs[kReadRows];
#pragma unroll
        for (int i = 0; i < kReadRows; i++) {
            if (i < rows && row_at[i] >= 0) {
                const int64_t e = row_at[i] + (int64_t)h * page * D + d, se = scale_at[i] + h * (page / kKv8Block);
                kw[i] = *reinterpret_cast<const uint32_t *>(p.pool.k + e);
                vw[i] = *reinterpret_cast<const uint32_t *>(p.pool.v + e);
                ks[i] = p.pool.ks[se], vs[i] = p.pool.vs[se];
            } else {
                kw[i] = vw[i] = 0;
                ks[i] = vs[i] = __int_as_float(0x7fc00000);
            }
        }
#pragma unroll
        for (int i = 0; i < kReadRows; i++) {
            if (i >= rows) break;
            float kx[4], vx[4];
            const uint32_t kb = kv8_unsign<E4M3>(kw[i]), vb = kv8_unsign<E4M3>(vw[i]);
            const uint32_t w[4] = {kv8_widen<E4M3, false>(kb), kv8_widen<E4M3, true>(kb), kv8_widen<E4M3, false>(vb),
                                   kv8_widen<E4M3, true>(vb)};
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&w[u]));
                const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&w[2 + u]));
                kx[2 * u] = a.x * ks[i], kx[2 * u + 1] = a.y * ks[i];
                vx[2 * u] = b.x * vs[i], vx[2 * u + 1] = b.y * vs[i];
            }
            const int64_t o = (r0 + i) * width * 4 + x * 4;
            if (p.k_out) store_act<T, 4>(static_cast<T *>(p.k_out) + o, kx, true);
            if (p.v_out) store_act<T, 4>(static_cast<T *>(p.v_out) + o, vx, true);
        }
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

static int64_t append_max_blocks(const vkq_kv8_batch &b) { return (b.max_tokens + kKv8Block - 2) / kKv8Block + 1; }
int64_t kv8_append_ctas(const vkq_kv8_cache &c, const vkq_kv8_batch &b, bool q) {
    return b.batch * append_max_blocks(b) * c.kv_heads * 2 + (q ? b.tokens : 0);
}

cudaError_t kv8_append(const vkq_kv8_cache &c, int64_t layer, const vkq_kv8_batch &b, const Kv8AppendArgs &a,
                       cudaStream_t s, int device) {
    AppendParams p{};
    p.pool = kv8_pool(c, layer);
    p.batch = kv8_batch(b);
    p.k = a.k, p.v = a.v, p.q = a.q, p.q_out = a.q_out;
    p.kt = a.k_token, p.vt = a.v_token, p.qt = a.q_token, p.qot = a.q_out_token;
    p.cos_t = a.cos_t, p.sin_t = a.sin_t, p.max_seq = a.max_seq;
    p.heads = (int)a.heads, p.rot = (int)a.rot_dim, p.half = a.layout == VKQ_ROPE_HALF;
    p.max_blocks = (uint32_t)append_max_blocks(b);
    // Where the new tokens' blocks alone are half of what the card holds (six CTAs
    // an SM), a CTA takes all items of its block: one look-up, the next item's
    // rows under way.  Fewer are spread, an item a CTA.  Measured, all / one, 8
    // KV heads in bfloat16 with q's 40: 9,472 tokens 75 / 102 us, 4,736 tokens 64
    // / 53, 1,024 tokens 34 / 18, 64 tokens 32 / 5.
    const bool many = b.tokens / kKv8Block >= 3 * device_sm_count(device);
    p.items = many ? 2 * c.kv_heads : 1;
    p.groups = (uint32_t)((2 * c.kv_heads + p.items - 1) / p.items);
    p.block_ctas = (uint32_t)(b.batch * p.max_blocks * p.groups);
    p.magic_groups = kv8_magic(p.groups), p.magic_blocks = kv8_magic(p.max_blocks);
    p.magic_page = kv8_magic((uint32_t)(c.page_size / kKv8Block));
    // a lane's D / 32 values as one vector
    const int size = act_bytes(a.dtype);
    const uintptr_t lane = (uintptr_t)(c.head_dim / 32 * size) - 1;
    p.vec_kv = (((uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)(a.k_token * size) | (uintptr_t)(a.v_token * size)) & lane) == 0;
    p.vec_t = (((uintptr_t)a.cos_t | (uintptr_t)a.sin_t) & 15u) == 0 && a.rot_dim % 8 == 0;
    int64_t ctas = p.block_ctas;
    if (a.q) {
        const uintptr_t bits = (uintptr_t)a.q | (uintptr_t)a.q_out | (uintptr_t)a.cos_t | (uintptr_t)a.sin_t |
                               (uintptr_t)(a.q_token * size) | (uintptr_t)(a.q_out_token * size);
        p.vec_q = rotary_vec(bits, a.rot_dim);
        const int pieces = size == 4 ? rotary_pieces<float>(c.head_dim, p.rot, p.half)
                                     : rotary_pieces<__half>(c.head_dim, p.rot, p.half);
        p.q_items = p.vec_q ? (p.heads + kRotHeads - 1) / kRotHeads * pieces : p.heads * (c.head_dim - p.rot / 2);
        // many tokens share the search for their sequence; few are spread (one
        // sequence, shared / alone: 9,472 tokens 75 / 79 us, 2,368 tokens 33 / 27)
        p.q_tokens = many ? kAppMaxTokens : 1;
        ctas += (b.tokens + p.q_tokens - 1) / p.q_tokens;
    }
    const void *fn = a.dtype == VKQ_F32   ? append_fn<float>(c.head_dim)
                     : a.dtype == VKQ_F16 ? append_fn<__half>(c.head_dim)
                                          : append_fn<__nv_bfloat16>(c.head_dim);
    return launch(fn, ctas, kAppThreads, &p, s);
}

template <typename T>
static const void *read_fn(bool e4m3) {
    return e4m3 ? (const void *)read_kernel<T, true> : (const void *)read_kernel<T, false>;
}

cudaError_t kv8_read(const vkq_kv8_cache &c, int64_t layer, const vkq_kv8_batch &b, const int *seq, const int *pos,
                     int64_t n, int dtype, void *k_out, void *v_out, cudaStream_t s) {
    ReadParams p{};
    p.pool = kv8_pool(c, layer);
    p.batch = kv8_batch(b);
    p.seq = seq, p.pos = pos, p.n = n, p.k_out = k_out, p.v_out = v_out;
    // rows of a CTA, kReadRows / 1, 8 heads to bfloat16: 256 rows 4.4 / 3.0 us,
    // 1,024 rows 4.6 / 5.3, 16,384 rows 33 / 71 (3.1 TB/s)
    p.rows = n >= 1024 ? kReadRows : 1;
    const void *fn = dtype == VKQ_F32   ? read_fn<float>(p.pool.e4m3)
                     : dtype == VKQ_F16 ? read_fn<__half>(p.pool.e4m3)
                                        : read_fn<__nv_bfloat16>(p.pool.e4m3);
    return launch(fn, (n + p.rows - 1) / p.rows, kReadThreads, &p, s);
}

int *kv8_status_word() { return status_word(g_kv8_status); }

}  // namespace vkq
