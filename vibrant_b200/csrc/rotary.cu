// rotary.cu -- rotary positions over strided [tokens][heads][head_dim]
// activations (both pair layouts, part of the head, f32/f16/bf16), and the
// cos/sin tables with the scalings for long contexts.
//
// A pair (x_a, x_b) of a head at position p turns by the table entry (c, s) of
// p: out_a = x_a c - x_b s, out_b = x_a s + x_b c.  One read and one write of
// the rotated heads, so HBM bounds it: a thread takes the 16-byte pieces that
// hold one group of pairs (one piece with interleaved pairs, the two partner
// pieces with half pairs) and keeps their c and s in registers for up to
// kRotHeads heads of the token, because reading them again for every head
// would be as many bytes from L1 as the heads themselves.
#include <cmath>
#include <cstdint>

#include "../../include/vkq.h"
#include "act.cuh"
#include "kq_device.cuh"
#include "vkq_internal.h"

namespace vkq {

static __device__ int g_rotary_status;

constexpr int kRotThreads = 128;
constexpr int kRotHeads = 4;

struct RotaryParams {
    const void *x;
    void *out;
    const float *cos_t, *sin_t;
    const int *pos;
    int64_t xt, xh, ot, oh;  // token and head strides, in elements
    int64_t items, max_seq;
    int heads, D, rot, pieces, groups;  // pieces of a head, groups of kRotHeads heads
    bool half, inverse;
};

// N pairs' table entries; aligned because N divides rot / 2 or the row is read one by one.
template <int N>
__device__ __forceinline__ void load_table(const float *t, float (&r)[N], bool vec) {
    load_act<float, N>(t, r, vec);
}

// The vector path: heads in 16-byte pieces of V elements, rot a multiple of
// 2V, aligned rows.  Interleaved: piece j of D / V (the rotated ones first);
// half: the rot / 2V partner pairs, then the pieces past rot.
template <typename T, bool HALF>
__global__ void __launch_bounds__(kRotThreads) rotary_vec_kernel(const RotaryParams p) {
    constexpr int V = 16 / (int)sizeof(T);
    constexpr int NP = HALF ? V : V / 2;  // pairs of an item
    pdl_wait();
    pdl_launch_dependents();
    const int64_t stride = (int64_t)gridDim.x * kRotThreads;
    for (int64_t it = (int64_t)blockIdx.x * kRotThreads + threadIdx.x; it < p.items; it += stride) {
        const int64_t tg = it / p.pieces;
        const int j = (int)(it - tg * p.pieces);
        const int64_t t = tg / p.groups;
        const int h0 = (int)(tg - t * p.groups) * kRotHeads;
        const int ps = p.pos[t];
        if (ps < 0 || ps >= p.max_seq) {
            atomicExch(&g_rotary_status, VKQ_ERR_INVALID_ARGUMENT);
            continue;
        }
        const int turned = HALF ? p.rot / (2 * V) : p.rot / V;
        const bool turns = j < turned;
        // first element of the piece, and of its partner
        const int a0 = HALF && !turns ? p.rot + (j - turned) * V : j * V;
        const int b0 = HALF ? a0 + p.rot / 2 : a0;
        float c[NP], s[NP];
        if (turns) {
            const int64_t e = (int64_t)ps * (p.rot / 2) + (HALF ? a0 : a0 / 2);
            // entries start at a multiple of 4 floats when rot is a multiple of 2V and V of 8, of 2 for V = 4 interleaved
            load_table<NP>(p.cos_t + e, c, true);
            load_table<NP>(p.sin_t + e, s, true);
            if (p.inverse)
#pragma unroll
                for (int i = 0; i < NP; i++) s[i] = -s[i];
        }
        const T *x = static_cast<const T *>(p.x) + t * p.xt;
        T *o = static_cast<T *>(p.out) + t * p.ot;
        float a[kRotHeads][V], b[kRotHeads][V];
#pragma unroll
        for (int u = 0; u < kRotHeads; u++) {
            if (h0 + u >= p.heads) break;
            const T *xh = x + (h0 + u) * p.xh;
            load_act<T, V>(xh + a0, a[u], true);
            if (HALF && turns) load_act<T, V>(xh + b0, b[u], true);
        }
#pragma unroll
        for (int u = 0; u < kRotHeads; u++) {
            if (h0 + u >= p.heads) break;
            if (turns) {
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    if constexpr (HALF) turn(a[u][i], b[u][i], c[i], s[i]);
                    else turn(a[u][2 * i], a[u][2 * i + 1], c[i], s[i]);
                }
            }
            T *oh = o + (h0 + u) * p.oh;
            store_act<T, V>(oh + a0, a[u], true);
            if (HALF && turns) store_act<T, V>(oh + b0, b[u], true);
        }
    }
}

// Any rot, strides and alignment: an item is one pair, or one value past rot.
template <typename T>
__global__ void __launch_bounds__(kRotThreads) rotary_any_kernel(const RotaryParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int half = p.rot / 2;
    const int64_t stride = (int64_t)gridDim.x * kRotThreads;
    for (int64_t it = (int64_t)blockIdx.x * kRotThreads + threadIdx.x; it < p.items; it += stride) {
        const int64_t th = it / p.pieces;
        const int j = (int)(it - th * p.pieces);
        const int64_t t = th / p.heads, h = th - t * p.heads;
        const int ps = p.pos[t];
        if (ps < 0 || ps >= p.max_seq) {
            atomicExch(&g_rotary_status, VKQ_ERR_INVALID_ARGUMENT);
            continue;
        }
        const T *x = static_cast<const T *>(p.x) + t * p.xt + h * p.xh;
        T *o = static_cast<T *>(p.out) + t * p.ot + h * p.oh;
        if (j >= half) {
            o[half + j] = x[half + j];
            continue;
        }
        const int ia = p.half ? j : 2 * j, ib = p.half ? j + half : 2 * j + 1;
        const int64_t e = (int64_t)ps * half + j;
        float a = to_f32<T>(x[ia]), b = to_f32<T>(x[ib]);
        const float s = p.sin_t[e];
        turn(a, b, p.cos_t[e], p.inverse ? -s : s);
        o[ia] = from_f32<T>(a);
        o[ib] = from_f32<T>(b);
    }
}

struct TableParams {
    float *cos_t, *sin_t;
    int64_t entries;
    int half;
    double step;       // t_i = exp(i * step), step = -2 ln(base') / rot
    double inv_factor; // the interpolated part's factor
    double low, width; // w_i = clamp((i - low) / width, 0, 1); width 0: w_i = 1
    double mscale;
};

__global__ void __launch_bounds__(256) rotary_tables_kernel(const TableParams p) {
    pdl_wait();
    pdl_launch_dependents();
    for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < p.entries;
         e += (int64_t)gridDim.x * blockDim.x) {
        const int64_t ps = e / p.half;
        const double i = (double)(e - ps * p.half);
        const double t = exp(i * p.step);
        const double w = p.width > 0 ? fmin(fmax((i - p.low) / p.width, 0.0), 1.0) : 1.0;
        const double f = t * p.inv_factor * w + t * (1.0 - w);
        double s, c;
        sincos((double)ps * f, &s, &c);
        p.cos_t[e] = (float)(c * p.mscale);
        p.sin_t[e] = (float)(s * p.mscale);
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
static const void *rotary_fn(bool vec, bool half) {
    if (!vec) return (const void *)rotary_any_kernel<T>;
    return half ? (const void *)rotary_vec_kernel<T, true> : (const void *)rotary_vec_kernel<T, false>;
}

cudaError_t rotary(const RotaryArgs &a, cudaStream_t s, int device) {
    const int size = act_bytes(a.dtype), V = 16 / size;
    RotaryParams p{};
    p.x = a.x, p.out = a.out, p.cos_t = a.cos_t, p.sin_t = a.sin_t, p.pos = a.positions;
    p.xt = a.x_token, p.xh = a.x_head, p.ot = a.out_token, p.oh = a.out_head;
    p.max_seq = a.max_seq;
    p.heads = (int)a.heads, p.D = (int)a.head_dim, p.rot = (int)a.rot_dim;
    p.half = a.layout == VKQ_ROPE_HALF, p.inverse = a.inverse != 0;
    // 16-byte pieces: whole ones in every row, pairs (and partners) whole pieces apart
    const uintptr_t bits = (uintptr_t)a.x | (uintptr_t)a.out | (uintptr_t)a.cos_t | (uintptr_t)a.sin_t |
                           (uintptr_t)((a.x_token | a.x_head | a.out_token | a.out_head | a.head_dim) * size);
    const bool vec = (bits & 15u) == 0 && a.rot_dim % 16 == 0;
    if (vec) {
        p.pieces = p.half ? p.rot / (2 * V) + (p.D - p.rot) / V : p.D / V;
        p.groups = (p.heads + kRotHeads - 1) / kRotHeads;
        p.items = a.tokens * p.groups * p.pieces;
    } else {
        p.pieces = p.D - p.rot / 2;
        p.items = a.tokens * p.heads * p.pieces;
    }
    int64_t blocks = (p.items + kRotThreads - 1) / kRotThreads;
    const int64_t cap = 64 * (int64_t)device_sm_count(device);
    if (blocks > cap) blocks = cap;
    const void *fn = a.dtype == VKQ_F32   ? rotary_fn<float>(vec, p.half)
                     : a.dtype == VKQ_F16 ? rotary_fn<__half>(vec, p.half)
                                          : rotary_fn<__nv_bfloat16>(vec, p.half);
    return launch(fn, blocks, kRotThreads, &p, s);
}

cudaError_t rotary_tables(float *cos_t, float *sin_t, int64_t max_seq, int64_t rot_dim, double base, int scaling,
                          double factor, int64_t orig_len, double beta_fast, double beta_slow, double attn_factor,
                          cudaStream_t s, int device) {
    TableParams p{};
    p.cos_t = cos_t, p.sin_t = sin_t;
    p.half = (int)(rot_dim / 2);
    p.entries = max_seq * p.half;
    const double r = (double)rot_dim;
    if (scaling == VKQ_ROPE_SCALE_NTK) base *= std::pow(factor, r / (r - 2.0));
    p.step = -2.0 * std::log(base) / r;
    p.inv_factor = scaling == VKQ_ROPE_SCALE_LINEAR || scaling == VKQ_ROPE_SCALE_YARN ? 1.0 / factor : 1.0;
    p.mscale = 1.0;
    if (scaling == VKQ_ROPE_SCALE_YARN) {
        const double pi = 3.14159265358979323846;
        auto at = [&](double beta) { return r * std::log((double)orig_len / (2.0 * pi * beta)) / (2.0 * std::log(base)); };
        const double top = r / 2.0 - 1.0;
        p.low = std::fmin(std::fmax(std::floor(at(beta_fast)), 0.0), top);
        const double high = std::fmin(std::fmax(std::ceil(at(beta_slow)), 0.0), top);
        p.width = std::fmax(high - p.low, 1e-3);  // equal ends: a step
        p.mscale = attn_factor > 0 ? attn_factor : 0.1 * std::log(factor) + 1.0;
    }
    int64_t blocks = (p.entries + 255) / 256;
    const int64_t cap = 16 * (int64_t)device_sm_count(device);
    if (blocks > cap) blocks = cap;
    return launch((const void *)rotary_tables_kernel, blocks, 256, &p, s);
}

int rotary_read_status() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_rotary_status, sizeof(int)) != cudaSuccess) return -1;
    cudaMemcpyToSymbol(g_rotary_status, &zero, sizeof(int));
    return v;
}

}  // namespace vkq
