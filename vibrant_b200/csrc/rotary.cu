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
// would be as many bytes from L1 as the heads themselves.  8,191 tokens of 40
// heads of 128, whole rows: 26 us in bfloat16 interleaved (6.3 TB/s), 33 halved,
// 52 in float32 (6.5 TB/s).  Rows or rot_dim that are no whole pieces go value by
// value, a pair a thread with entries of its own: 119 us, left so as the rarer
// case.  One token 2 us either way.
#include <cmath>
#include <cstdint>

#include "../../include/vkq.h"
#include "act.cuh"
#include "kq_device.cuh"
#include "rotary.cuh"
#include "vkq_internal.h"

namespace vkq {

static __device__ int g_rotary_status;

constexpr int kRotThreads = 128;

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

template <typename T, bool HALF, typename I>
__global__ void __launch_bounds__(kRotThreads) rotary_vec_kernel(const RotaryParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const I items = (I)p.items, stride = (I)gridDim.x * kRotThreads;
    for (I it = (I)blockIdx.x * kRotThreads + threadIdx.x; it < items; it += stride) {
        const I tg = it / (I)p.pieces;
        const int j = (int)(it - tg * (I)p.pieces);
        const I t = tg / (I)p.groups;
        const int h0 = (int)(tg - t * (I)p.groups) * kRotHeads;
        const int ps = p.pos[t];
        rotary_item<T, HALF>(static_cast<const T *>(p.x) + (int64_t)t * p.xt + h0 * p.xh, p.xh,
                             static_cast<T *>(p.out) + (int64_t)t * p.ot + h0 * p.oh, p.oh, p.heads - h0, j, p.D, p.rot,
                             p.cos_t, p.sin_t, p.inverse, [&]() -> int64_t {
                                 if (ps >= 0 && ps < p.max_seq) return ps;
                                 atomicExch(&g_rotary_status, VKQ_ERR_INVALID_ARGUMENT);
                                 return -1;
                             });
    }
}

template <typename T>
__global__ void __launch_bounds__(kRotThreads) rotary_any_kernel(const RotaryParams p) {
    pdl_wait();
    pdl_launch_dependents();
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
        rotary_one<T>(static_cast<const T *>(p.x) + t * p.xt + h * p.xh, static_cast<T *>(p.out) + t * p.ot + h * p.oh, j,
                      p.rot, p.half, p.cos_t, p.sin_t, p.inverse, ps);
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
static const void *rotary_fn(bool vec, bool half, bool small) {
    if (!vec) return (const void *)rotary_any_kernel<T>;
    if (small)
        return half ? (const void *)rotary_vec_kernel<T, true, uint32_t> : (const void *)rotary_vec_kernel<T, false, uint32_t>;
    return half ? (const void *)rotary_vec_kernel<T, true, int64_t> : (const void *)rotary_vec_kernel<T, false, int64_t>;
}

cudaError_t rotary(const RotaryArgs &a, cudaStream_t s, int device) {
    const int size = act_bytes(a.dtype);
    RotaryParams p{};
    p.x = a.x, p.out = a.out, p.cos_t = a.cos_t, p.sin_t = a.sin_t, p.pos = a.positions;
    p.xt = a.x_token, p.xh = a.x_head, p.ot = a.out_token, p.oh = a.out_head;
    p.max_seq = a.max_seq;
    p.heads = (int)a.heads, p.D = (int)a.head_dim, p.rot = (int)a.rot_dim;
    p.half = a.layout == VKQ_ROPE_HALF, p.inverse = a.inverse != 0;
    // 16-byte pieces: whole ones in every row, pairs (and partners) whole pieces apart
    const uintptr_t bits = (uintptr_t)a.x | (uintptr_t)a.out | (uintptr_t)a.cos_t | (uintptr_t)a.sin_t |
                           (uintptr_t)((a.x_token | a.x_head | a.out_token | a.out_head | a.head_dim) * size);
    const bool vec = rotary_vec(bits, a.rot_dim);
    if (vec) {
        p.pieces = size == 4 ? rotary_pieces<float>(p.D, p.rot, p.half) : rotary_pieces<__half>(p.D, p.rot, p.half);
        p.groups = (p.heads + kRotHeads - 1) / kRotHeads;
        p.items = a.tokens * p.groups * p.pieces;
    } else {
        p.pieces = p.D - p.rot / 2;
        p.items = a.tokens * p.heads * p.pieces;
    }
    int64_t blocks = (p.items + kRotThreads - 1) / kRotThreads;
    const int64_t cap = 64 * (int64_t)device_sm_count(device);
    if (blocks > cap) blocks = cap;
    const bool small = p.items + blocks * kRotThreads < (int64_t(1) << 32);  // 32-bit item numbers
    const void *fn = a.dtype == VKQ_F32   ? rotary_fn<float>(vec, p.half, small)
                     : a.dtype == VKQ_F16 ? rotary_fn<__half>(vec, p.half, small)
                                          : rotary_fn<__nv_bfloat16>(vec, p.half, small);
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
        const double top = r - 1.0;  // the definition's limit: a ramp may end past the last pair, r / 2 - 1
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

int *rotary_status_word() { return status_word(g_rotary_status); }

}  // namespace vkq
