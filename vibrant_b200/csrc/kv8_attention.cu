// kv8_attention.cu -- attention of few query rows over the 8-bit paged KV
// cache (decode steps, verified proposals, short chunks).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp2(f ks_j (q . ck_j) - m)
// with f = scale log2(e), codes ck, cv and block scales ks, vs.  The rows of a
// tile are the (new token, query head) pairs of one sequence and KV head, so
// that the heads of a group share one read of the cache; that read bounds a
// decode step (2 (D + 1/4) bytes a cached token and KV head).
//
// A CTA takes one tile and one range of keys; its four warps take steps of 32
// keys in turn, each through a ring of its own filled by 16-byte cp.async, and
// keep a running maximum, sum and output, joined in shared memory at the end.
// The ranges are joined by the CTA of the tile that finishes last, in range
// order, so results do not depend on timing.
//
// The products run on m16n8k16 with float16 operands: codes are exact in
// float16 (kv8_widen), and a decode step has some 16 rows, which leave a
// 128-row tcgen05 tile with q's rows in it nearly empty (many_rows has both
// sides measured; the operands exchanged, keys in the 128 rows and q's rows as
// columns, would fill it and have not been built).  Each
// lane's operand columns are chosen so that its 16-byte loads from shared memory
// hold whole fragments: column k of a K step is dimension 16 (c + 4 h) + 4 w +
// ..., column n of a V tile t is dimension (D / 8) n + t; the same order on both
// sides of a product, so it drops out.
//
// Measured, 40 heads on 8 of D = 128: one context of 200,001 tokens in float32
// 93 us (4.4 TB/s), 32 of 500 to 9,000 in bfloat16 56 us (3.3 TB/s); one token of
// 1,024 with 16 heads on 2 9 us, a chain of latencies.  The longer ones are bound
// by the instructions that turn codes into operands, behind them by the loads of
// two-deep rings: 146 us with two CTAs an SM and 16-row tiles for eight rows.
//
// Precision.  float32 q and p are split, x = hi + lo with two float16 parts
// (22 bits), one product each: with 8 rows the parts are rows r and r + 8 of
// one instruction, so the split costs nothing there.  q is first scaled by a
// power of two of its row, and p by 2^14, to keep the low parts out of
// float16's subnormals.  16-bit q is exact in float16 after that scaling; with
// more than 8 rows its p is rounded once to 11 bits (2^-11, no more than the
// output's own rounding) and the tile has 16 rows.  Each 16-key product starts from zero and is
// added to the output in float32 with its vs: the accumulators of the matrix
// unit round toward zero, which would add up over a long cache.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../../include/vkq.h"
#include "act.cuh"
#include "kq_device.cuh"
#include "kv8.cuh"
#include "vkq_internal.h"

namespace vkq {

static __device__ int g_kv8_attn_status;

constexpr int kDecWarps = 4;
constexpr int kDecThreads = 32 * kDecWarps;
constexpr int kDecStep = 32;   // keys of a step: two scale blocks
constexpr int kDecStages = 2;  // ring slots of a warp
// CTAs an SM that registers and rings are cut for (16 rows take the registers of two)
constexpr int dec_ctas(int rows) { return rows == 8 ? 3 : 2; }

struct DecodeParams {
    Kv8Pool pool;
    Kv8Batch batch;
    const void *q;
    void *out;
    int64_t qt, ot;
    int heads, g, row_tiles, splits, chunk;
    uint32_t magic;  // of page / 16 (kv8_div)
    float f;      // scale * log2(e)
    int causal, window;
    bool vec;     // rows of q and out are 16-byte aligned
    float *part;  // [tile][split][rows][D], then [tile][split][rows][2]
    float *stat;
    unsigned *count;  // a tile's finished ranges; zero before and after a call
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 half2_floats(uint32_t b) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&b));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same from zero.
__device__ __forceinline__ void mma_f16_new(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// The sum over a warp's lanes, the same in each.
__device__ __forceinline__ float warp_total(float s) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// Byte offset of 16-byte piece `ch` of row r (of 16) in a ring slot, permuted
// so that the K reads (two rows, four pieces) and the V reads (four even or
// odd rows, two pieces) of eight lanes fall into different banks.
template <int D>
__device__ __forceinline__ uint32_t slot_off(int r, int ch) {
    if constexpr (D == 128) return (uint32_t)(r * 128 + ((ch ^ ((r & 6) ^ ((r & 1) << 2))) << 4));
    else return (uint32_t)((r >> 1) * 128 + (((((r & 1) << 2) | ch) ^ (((r >> 1) & 3) << 1)) << 4));
}

template <typename T, int D, bool E4M3, int ROWS>
__global__ void __launch_bounds__(kDecThreads, dec_ctas(ROWS)) kv8_decode_kernel(const DecodeParams p) {
    // Eight rows leave the instruction's other eight to the low parts (of 16-bit
    // q: zeros); sixteen 16-bit rows are rounded.
    constexpr bool SPLIT = ROWS == 8;
    static_assert(SPLIT || sizeof(T) == 2, "float32 takes both parts");
    constexpr int NR = ROWS / 8;  // rows of a lane
    constexpr int KS = D / 16;                                // K steps
    constexpr int NT = D / 8;                                 // V tiles
    constexpr int UNIT = kKv8Block * D;                       // code bytes of 16 keys
    constexpr int SLOT = 4 * UNIT + 16;                       // a step: K and V of two units, four scales
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ bool last;
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n8 = lane >> 2, c = lane & 3;
    const int rt = blockIdx.x / p.splits, split = blockIdx.x - rt * p.splits, kvh = blockIdx.y;
    const Kv8Seq s = kv8_seq(p.batch, p.pool.page, blockIdx.z);
    const int rows_all = s.n * p.g;
    const int r0 = rt * ROWS;
    if (!s.ok) {
        if (split > 0) return;
        if (threadIdx.x == 0) atomicExch(&g_kv8_attn_status, VKQ_ERR_INVALID_ARGUMENT);
        for (int i = threadIdx.x; i < ROWS * D; i += kDecThreads) {
            const int r = r0 + i / D;
            if (r < rows_all)
                static_cast<T *>(p.out)[(int64_t)(s.first + r / p.g) * p.ot + (int64_t)(kvh * p.g + r % p.g) * D + i % D] =
                    from_f32<T>(__int_as_float(0x7fc00000));
        }
        return;
    }
    if (r0 >= rows_all) return;
    // the keys that the tile's rows can see, from a block's first
    const int pos0 = s.len - s.n;
    const int row_end = min(r0 + ROWS, rows_all) - 1;
    const int hi = p.causal ? max(pos0 + row_end / p.g + 1, 0) : s.len;
    int lo = 0;
    if (p.window > 0) lo = max(pos0 + r0 / p.g - p.window + 1, 0) & ~(kKv8Block - 1);
    const int active = max((hi - lo + p.chunk - 1) / p.chunk, 1);
    if (split >= active) return;
    const int k_lo = lo + split * p.chunk, k_hi = min(hi, k_lo + p.chunk);

    // the warp's ring
    const uint32_t my_ring = smem_u32addr(ring) + (uint32_t)(warp * kDecStages * SLOT);
    const int steps = k_hi > k_lo ? (k_hi - k_lo + kDecStep - 1) / kDecStep : 0;
    const int mine = steps > warp ? (steps - warp + kDecWarps - 1) / kDecWarps : 0;
    bool bad = false;
    const uint32_t per_page = (uint32_t)(p.pool.page / kKv8Block);
    const int lrow = lane / (D / 16), lch = lane % (D / 16);   // the lane's first piece; the next are LSTEP rows on
    constexpr int LSTEP = 32 / (D / 16), PIECES = UNIT / 512;  // 4 rows, 4 pieces (D = 64: 8, 2)
    uint32_t loff[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; i++) loff[i] = slot_off<D>(lrow + i * LSTEP, lch);
    auto fill = [&](int it) {
        if (it < mine) {
            const uint32_t slot = my_ring + (uint32_t)(it % kDecStages) * SLOT;
            const int key = k_lo + (warp + it * kDecWarps) * kDecStep;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int k0 = key + u * kKv8Block;
                // the unit's block in the layer's pool ([page][kv head][block]), 0 where there is none
                int id = -1;
                uint32_t blk = (uint32_t)k0 / kKv8Block;
                if (k0 < k_hi) {
                    const uint32_t lp = kv8_div(blk, per_page, p.magic);
                    id = kv8_page(p.pool, s, (int)lp);
                    bad |= id < 0;
                    blk -= lp * per_page;
                }
                const int rows = id < 0 ? 0 : min(k_hi - k0, kKv8Block);
                const int64_t b = id < 0 ? 0 : ((int64_t)id * p.pool.kv_heads + kvh) * per_page + blk;
                const uint8_t *ks = p.pool.k + b * UNIT + lane * 16, *vs = p.pool.v + b * UNIT + lane * 16;
                const uint32_t kd = slot + (uint32_t)(u * UNIT), vd = slot + (uint32_t)((2 + u) * UNIT);
#pragma unroll
                for (int i = 0; i < PIECES; i++) {  // rows past the range are zeros
                    const uint32_t bytes = lrow + i * LSTEP < rows ? 16u : 0u;
                    cp_async16(kd + loff[i], ks + i * 512, bytes);
                    cp_async16(vd + loff[i], vs + i * 512, bytes);
                }
                if (lane < 2)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(slot + 4u * UNIT + 8u * u + 4u * lane),
                                 "l"((lane ? p.pool.vs : p.pool.ks) + b), "r"(id < 0 ? 0u : 4u)
                                 : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    // the first steps are under way while q is loaded
#pragma unroll
    for (int it = 0; it < kDecStages - 1; it++) fill(it);

    // q: the lane's rows (n8, and n8 + 8 with 16-bit rows), scaled to below 2^15
    uint32_t qa[KS][4];
    float rf[NR];          // what a score of the row is multiplied by, with ks
    int see_lo[NR], see_hi[NR];
#pragma unroll
    for (int u = 0; u < NR; u++) {
        const int r = r0 + n8 + 8 * u;
        const bool there = r < rows_all;
        const int i = there ? r / p.g : 0, h = kvh * p.g + (there ? r % p.g : 0);
        const int ps = pos0 + i;
        see_hi[u] = !there ? 0 : p.causal ? ps + 1 : s.len;
        see_lo[u] = p.window > 0 ? ps - p.window + 1 : 0;
        const T *q = static_cast<const T *>(p.q) + (int64_t)(s.first + i) * p.qt + (int64_t)h * D;
        float x[D / 64][16];
        float a = 0.f;
#pragma unroll
        for (int hh = 0; hh < D / 64; hh++) {
            load_act<T, 16>(q + 16 * (c + 4 * hh), x[hh], p.vec);
#pragma unroll
            for (int t = 0; t < 16; t++) a = fmaxf(a, fabsf(x[hh][t]));
        }
        a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
        a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
        const int e = min(max((int)(__float_as_uint(a) >> 23) - 127, -60), 127);
        const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23);
        rf[u] = p.f * __uint_as_float((uint32_t)(e - 14 + 127) << 23);
#pragma unroll
        for (int hh = 0; hh < D / 64; hh++)
#pragma unroll
            for (int w = 0; w < 4; w++)
#pragma unroll
                for (int z = 0; z < 2; z++) {
                    const float x0 = x[hh][4 * w + 2 * z] * up, x1 = x[hh][4 * w + 2 * z + 1] * up;
                    const uint32_t b = half2_bits(x0, x1);
                    if constexpr (SPLIT) {
                        const float2 back = half2_floats(b);
                        qa[4 * hh + w][2 * z] = b;
                        qa[4 * hh + w][2 * z + 1] = half2_bits(x0 - back.x, x1 - back.y);
                    } else {
                        qa[4 * hh + w][2 * z + u] = b;
                    }
                }
    }

    float m[NR], l[NR];
    float2 o[NT][NR];
#pragma unroll
    for (int u = 0; u < NR; u++) {
        m[u] = -INFINITY;
        l[u] = 0.f;
#pragma unroll
        for (int t = 0; t < NT; t++) o[t][u] = make_float2(0.f, 0.f);
    }
    for (int it = 0; it < mine; it++) {
        fill(it + kDecStages - 1);  // into the slot read one pass ago
        asm volatile("cp.async.wait_group %0;" ::"n"(kDecStages - 1) : "memory");
        __syncwarp();
        const uint32_t slot = my_ring + (uint32_t)(it % kDecStages) * SLOT;
        const int key = k_lo + (warp + it * kDecWarps) * kDecStep;
        const uint4 scw = lds128(slot + 4u * UNIT);  // ks, vs of unit 0; of unit 1
        const float ks[2] = {__uint_as_float(scw.x), __uint_as_float(scw.z)};
        const float vs[2] = {__uint_as_float(scw.y), __uint_as_float(scw.w)};

        float x[2][2][NR][2];  // scores: unit, 8-key tile, row, the lane's two keys
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                float d[4];
#pragma unroll
                for (int hh = 0; hh < D / 64; hh++) {
                    const uint4 kw = lds128(slot + (uint32_t)(u * UNIT) + slot_off<D>(8 * t + n8, c + 4 * hh));
                    const uint32_t w[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t b = kv8_unsign<E4M3>(w[i]);
                        if (hh == 0 && i == 0) mma_f16_new(d, qa[0], kv8_widen<E4M3, false>(b), kv8_widen<E4M3, true>(b));
                        else mma_f16(d, qa[4 * hh + i], kv8_widen<E4M3, false>(b), kv8_widen<E4M3, true>(b));
                    }
                }
                const int j = key + u * kKv8Block + 8 * t + 2 * c;
#pragma unroll
                for (int r = 0; r < NR; r++) {
                    const float f = ks[u] * rf[r];
#pragma unroll
                    for (int z = 0; z < 2; z++) {
                        const float raw = SPLIT ? d[z] + d[2 + z] : d[2 * r + z];
                        x[u][t][r][z] = j + z >= see_lo[r] && j + z < see_hi[r] && j + z < k_hi ? raw * f : -INFINITY;
                    }
                }
            }

        // the running maximum; p = 2^14 exp2(x - m)
        float alpha[NR];
        bool grew = false;
#pragma unroll
        for (int r = 0; r < NR; r++) {
            float a = m[r];
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int t = 0; t < 2; t++) a = fmaxf(a, fmaxf(x[u][t][r][0], x[u][t][r][1]));
            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
            const float base = a == -INFINITY ? 0.f : a;  // nothing visible yet
            alpha[r] = ex2(m[r] - base);
            grew |= a > m[r];
            m[r] = a;
            float sum = 0.f;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int z = 0; z < 2; z++) {
                        x[u][t][r][z] = ex2(x[u][t][r][z] - base + 14.f);
                        sum += x[u][t][r][z];
                    }
            l[r] = l[r] * alpha[r] + sum;
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const float2 al = make_float2(alpha[r], alpha[r]);
#pragma unroll
                for (int t = 0; t < NT; t++) o[t][r] = f2mul(o[t][r], al);
            }
        }

        // o += vs * (p . cv), 16 keys at a time
#pragma unroll
        for (int u = 0; u < 2; u++) {
            uint32_t pa[4];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                pa[2 * t] = half2_bits(x[u][t][0][0], x[u][t][0][1]);
                if constexpr (SPLIT) {
                    const float2 back = half2_floats(pa[2 * t]);
                    pa[2 * t + 1] = half2_bits(x[u][t][0][0] - back.x, x[u][t][0][1] - back.y);
                } else {
                    pa[2 * t + 1] = half2_bits(x[u][t][NR - 1][0], x[u][t][NR - 1][1]);
                }
            }
            const float sc = vs[u];
            const float2 sc2 = make_float2(sc, sc);
            const uint32_t vb = slot + (uint32_t)((2 + u) * UNIT);
            uint32_t w[4][NT / 4];  // the lane's dimensions of keys 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = 2 * c + (i & 1) + 8 * (i >> 1);
                if constexpr (D == 128) {
                    const uint4 t4 = lds128(vb + slot_off<D>(row, n8));
                    w[i][0] = t4.x, w[i][1] = t4.y, w[i][2] = t4.z, w[i][3] = t4.w;
                } else {
                    const uint2 t2 = lds64(vb + slot_off<D>(row, n8 >> 1) + 8u * (n8 & 1));
                    w[i][0] = t2.x, w[i][1] = t2.y;
                }
            }
#pragma unroll
            for (int i = 0; i < NT / 4; i++)
#pragma unroll
                for (int z = 0; z < 2; z++) {  // dimensions 4i + 2z, + 1: bytes of two keys side by side
                    const uint32_t b0 = kv8_unsign<E4M3>(prmt(w[0][i], w[1][i], z ? 0x7362u : 0x5140u));
                    const uint32_t b1 = kv8_unsign<E4M3>(prmt(w[2][i], w[3][i], z ? 0x7362u : 0x5140u));
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        float d[4];
                        if (y == 0) mma_f16_new(d, pa, kv8_widen<E4M3, false>(b0), kv8_widen<E4M3, false>(b1));
                        else mma_f16_new(d, pa, kv8_widen<E4M3, true>(b0), kv8_widen<E4M3, true>(b1));
                        const int t = 4 * i + 2 * z + y;
                        if constexpr (SPLIT) {
                            o[t][0] = f2fma(f2add(make_float2(d[0], d[1]), make_float2(d[2], d[3])), sc2, o[t][0]);
                        } else {
                            o[t][0] = f2fma(make_float2(d[0], d[1]), sc2, o[t][0]);
                            o[t][NR - 1] = f2fma(make_float2(d[2], d[3]), sc2, o[t][NR - 1]);
                        }
                    }
                }
        }
        __syncwarp();  // the slot may be filled again
    }
    asm volatile("cp.async.wait_all;" ::: "memory");

    // the four warps' parts, through shared memory (the rings are done with)
    const bool any_bad = __any_sync(0xffffffffu, bad);
    if (any_bad && lane == 0) atomicExch(&g_kv8_attn_status, VKQ_ERR_INVALID_ARGUMENT);
    __syncthreads();
    float *so = reinterpret_cast<float *>(ring);            // [warp][row][D]
    float *sm = so + kDecWarps * ROWS * D, *sl = sm + kDecWarps * ROWS;
#pragma unroll
    for (int r = 0; r < NR; r++) {
        float sum = l[r];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (any_bad) sum = __int_as_float(0x7fc00000);
        const int row = n8 + 8 * r;
        if (c == 0) sm[warp * ROWS + row] = m[r], sl[warp * ROWS + row] = sum;
        // column n of tile t is dimension NT n + t: the lane's two runs of NT
        float *d0 = so + (warp * ROWS + row) * D + 2 * c * NT;
#pragma unroll
        for (int t = 0; t < NT; t++) d0[t] = o[t][r].x, d0[NT + t] = o[t][r].y;
    }
    __syncthreads();
    const int64_t tile = ((int64_t)blockIdx.z * p.pool.kv_heads + kvh) * p.row_tiles + rt;
    float *part = p.part + (tile * p.splits + split) * ROWS * D;
    float *stat = p.stat + (tile * p.splits + split) * ROWS * 2;
    // four dimensions of a row a thread
    for (int i = threadIdx.x; i < ROWS * D / 4; i += kDecThreads) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float mx = sm[r];
#pragma unroll
        for (int w = 1; w < kDecWarps; w++) mx = fmaxf(mx, sm[w * ROWS + r]);
        float sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kDecWarps; w++) {
            const float mw = sm[w * ROWS + r], k = mw == -INFINITY ? 0.f : ex2(mw - mx);
            const float4 v = *reinterpret_cast<const float4 *>(so + (w * ROWS + r) * D + d);
            sum += k * sl[w * ROWS + r];
            acc[0] += k * v.x, acc[1] += k * v.y, acc[2] += k * v.z, acc[3] += k * v.w;
        }
        if (active > 1) {
            *reinterpret_cast<float4 *>(part + r * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
            if (d == 0) stat[2 * r] = mx, stat[2 * r + 1] = sum;
        } else if (r0 + r < rows_all) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
            for (int z = 0; z < 4; z++) acc[z] *= inv;
            store_act<T, 4>(static_cast<T *>(p.out) + (int64_t)(s.first + (r0 + r) / p.g) * p.ot +
                                (int64_t)(kvh * p.g + (r0 + r) % p.g) * D + d,
                            acc, p.vec);
        }
    }
    if (active == 1) return;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(p.count + tile, 1u) == (unsigned)active - 1u;
    __syncthreads();
    if (!last) return;
    __threadfence();
    if (threadIdx.x == 0) p.count[tile] = 0;
    part = p.part + tile * p.splits * ROWS * D;
    stat = p.stat + tile * p.splits * ROWS * 2;
    // each range's weight for each row, 1 / l folded in; then the sums, many loads in flight
    float *wt = reinterpret_cast<float *>(ring);  // [range][row]
    for (int r = warp; r < ROWS; r += kDecWarps) {
        float mx = -INFINITY, sum = 0.f;
        for (int w = lane; w < active; w += 32) mx = fmaxf(mx, __ldcg(stat + (w * ROWS + r) * 2));
#pragma unroll
        for (int i = 16; i > 0; i >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, i));
        for (int w = lane; w < active; w += 32) {
            const float2 ms = __ldcg(reinterpret_cast<const float2 *>(stat + (w * ROWS + r) * 2));
            const float k = ms.x == -INFINITY ? 0.f : ex2(ms.x - mx);
            sum += k * ms.y;
            wt[w * ROWS + r] = k;
        }
        sum = warp_total(sum);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        __syncwarp();
        for (int w = lane; w < active; w += 32) wt[w * ROWS + r] *= inv;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * D / 4; i += kDecThreads) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        if (r0 + r >= rows_all) continue;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        const float4 *v = reinterpret_cast<const float4 *>(part + (int64_t)r * D + d);
#pragma unroll 8
        for (int w = 0; w < active; w++) {
            const float4 x = __ldcg(v + (int64_t)w * (ROWS * D / 4));
            const float k = wt[w * ROWS + r];
            acc[0] += k * x.x, acc[1] += k * x.y, acc[2] += k * x.z, acc[3] += k * x.w;
        }
        store_act<T, 4>(static_cast<T *>(p.out) + (int64_t)(s.first + (r0 + r) / p.g) * p.ot +
                            (int64_t)(kvh * p.g + (r0 + r) % p.g) * D + d,
                        acc, p.vec);
    }
}

template <typename T, int D, int ROWS>
static const void *decode_fn(bool e4m3) {
    return e4m3 ? (const void *)kv8_decode_kernel<T, D, true, ROWS> : (const void *)kv8_decode_kernel<T, D, false, ROWS>;
}
template <typename T>
static const void *decode_fn(int D, bool e4m3, int rows) {
    if constexpr (sizeof(T) == 2)
        if (rows == 16) return D == 64 ? decode_fn<T, 64, 16>(e4m3) : decode_fn<T, 128, 16>(e4m3);
    return D == 64 ? decode_fn<T, 64, 8>(e4m3) : decode_fn<T, 128, 8>(e4m3);
}

// Keys that a tile of `rows` rows can see: all, or a window and the tile's own tokens.
static int64_t seen_keys(const vkq_kv8_batch &b, int64_t rows, int64_t g, int causal, int64_t window) {
    int64_t keys = b.max_len;
    if (causal && window > 0) {
        const int64_t w = window + (rows + g - 1) / g + kKv8Block;
        if (w < keys) keys = w;
    }
    return keys < 1 ? 1 : keys;
}

static Kv8Plan decode_plan(const vkq_kv8_cache &c, const vkq_kv8_batch &b, int dtype, int64_t heads, int causal,
                              int64_t window, int sms) {
    Kv8Plan q{};
    const int64_t g = heads / c.kv_heads;
    const int64_t keys = seen_keys(b, 16, g, causal, window);
    // 16-bit rows beyond eight: tiles of 16, which read the cache half as often,
    // where they have a step for each CTA that the card holds, else tiles of 8.
    // Measured in bfloat16, us in tiles of 8 / 16: 12 rows of 4,096 keys and 8 KV
    // heads 16.2 / 19.2 (256 steps of a CTA), 30 rows of 32,768 57.9 / 45.2, 15
    // rows of 32 contexts of 4,096 115 / 99.
    const int64_t rows = b.max_tokens * g, steps = b.batch * c.kv_heads * ((rows + 15) / 16) * ((keys + 127) / 128);
    q.rows = dtype == VKQ_F32 || rows <= 8 || steps < dec_ctas(16) * (int64_t)sms ? 8 : 16;
    q.row_tiles = (int)((rows + q.rows - 1) / q.rows);
    q.tiles = b.batch * c.kv_heads * q.row_tiles;
    // Ranges: what is cheapest in units of a CTA's round (a step of each warp),
    // over the CTAs that the card holds.  A CTA costs its rounds and kStart for
    // its start and end; each range of a tile kJoin more for the CTA that joins
    // them.  Several sequences, whose lengths the host does not know, are taken to
    // be kLong of max_len, and the last CTAs to be alone for kTail of their time
    // (31 of 500 to 9,000 with max_len 4 and 16 times the longest: 81, 85, 132 us).
    // (One sequence's ranges run at once: what is left is rounds / n + kJoin n.)
    // One range where the tiles are more than the workspace's head has counters
    // for.  Measured in bfloat16 with 8 KV heads, us in ranges of (most keys a
    // CTA): 3 contexts of 10,000 to 20,000 tokens 43 (384), 33 (1,024); 2 of 30,000
    // to 60,000 63 (768), 49 (1,440); 8 of 500 to 3,000 17 (256), 20 (512), 23
    // (1,024); 32 of 500 to 9,000 85 (4,608), 56 (1,800), 59 (1,500).
    constexpr double kStart = 3., kJoin = 0.1, kTail = 0.45, kLong = 0.7;
    const int64_t slots = dec_ctas(q.rows) * (int64_t)sms, steps_all = (keys + kDecStep - 1) / kDecStep;
    const int64_t most = (steps_all + kDecWarps - 1) / kDecWarps;
    int64_t best = 1;
    if (q.tiles <= kHeadCounters && b.batch == 1) {
        // all at once: least of most / n + kJoin n
        best = std::min(slots / q.tiles, (int64_t)std::sqrt((double)most / kJoin));
        best = std::max<int64_t>(1, std::min<int64_t>(best, std::min<int64_t>(most, 128)));
    } else if (q.tiles <= kHeadCounters) {
        double least = 0.;
        for (int64_t n = 1; n <= 128 && n <= most; n += 1 + n / 8) {
            const double rounds = (double)steps_all / (double)(kDecWarps * n), part = n > 1 ? kLong * (double)n : 1.;
            const double all = (double)q.tiles * ((double)most * kLong + kStart * part) / (double)slots + kTail * rounds;
            const double cost = std::max(rounds + kStart, all) + (n > 1 ? kJoin * (double)n : 0.);
            if (n == 1 || cost < least) best = n, least = cost;
        }
    }
    const int64_t chunk = ((keys + best - 1) / best + kDecStep - 1) / kDecStep * kDecStep;
    q.chunk = (int)chunk;
    q.splits = (int)((keys + chunk - 1) / chunk);
    if (q.splits > 1) {
        q.part_floats = (size_t)(q.tiles * q.splits * q.rows * c.head_dim);
        q.stat_floats = (size_t)(q.tiles * q.splits * q.rows * 2);
    }
    return q;
}

// Whether the 128-row tiles of kv8_prefill.cu pay: more than 32 rows of a
// sequence and KV head, and work for more than their 18 us of start and join.
// Measured, us here / there, bfloat16 (float32): 32 contexts of 4,096 keys and 8
// KV heads, 32 rows 166 / 185 (218 / 254), 64 rows 245 / 164 (378 / 229); one of
// 32,768, 20 rows 48 / 59 (50 / 77), 40 rows 63 / 58 (73 / 74), 80 rows 92 / 56
// (139 / 73); one of 2,048 and 2 KV heads, 64 rows 13 / 18 (14 / 18), 192 rows
// (786,432 pairs of a row and a key) 22 / 21 (16 / 18), 512 rows 25 / 21 (26 / 20).
// One rule for a call: single tokens beside a chunk take the chunk's tiles, and
// two calls are faster then.  One chunk of 512 and 31 tokens of 500 to 9,000, 40
// heads on 8: 256 (363) together, 54 + 81 (87 + 82) apart.
static bool many_rows(const vkq_kv8_cache &c, const vkq_kv8_batch &b, int64_t heads, int causal, int64_t window) {
    const int64_t g = heads / c.kv_heads, rows = b.max_tokens * g;
    const double pairs = (double)(rows * c.kv_heads * b.batch) * (double)seen_keys(b, rows, g, causal, window);
    return rows > 32 && pairs > (double)(1 << 19);
}

static Kv8Plan attention_plan(const vkq_kv8_cache &c, const vkq_kv8_batch &b, int dtype, int64_t heads, int causal,
                              int64_t window, int device) {
    const int sms = device_sm_count(device);
    return many_rows(c, b, heads, causal, window) ? kv8_prefill_plan(c, b, dtype, heads, causal, window, sms)
                                  : decode_plan(c, b, dtype, heads, causal, window, sms);
}

size_t kv8_attention_workspace(const vkq_kv8_cache &c, const vkq_kv8_batch &b, int dtype, int64_t heads, int causal,
                               int64_t window, int device, int64_t *ctas) {
    const Kv8Plan q = attention_plan(c, b, dtype, heads, causal, window, device);
    // (few rows: at most 2^16 tiles a sequence and head by many_rows, 128 ranges,
    // and the grid's other axes are held by the arguments' checks)
    *ctas = !many_rows(c, b, heads, causal, window) ? (int64_t)q.row_tiles * q.splits
            : q.splits == 1                         ? q.tiles
                                                    : q.tiles * std::max(q.splits, q.rows / 32);
    return kWorkspaceCounterHead + (q.part_floats + q.stat_floats) * sizeof(float);
}

cudaError_t kv8_attention(const vkq_kv8_cache &c, int64_t layer, const vkq_kv8_batch &b, const Kv8AttentionArgs &a,
                          cudaStream_t s, int device) {
    const Kv8Plan q = attention_plan(c, b, a.dtype, a.heads, a.causal, a.window, device);
    if (many_rows(c, b, a.heads, a.causal, a.window)) return kv8_prefill(c, layer, b, a, q, s);
    DecodeParams p{};
    p.pool = kv8_pool(c, layer);
    p.batch = kv8_batch(b);
    p.q = a.q, p.out = a.out, p.qt = a.q_token, p.ot = a.out_token;
    p.heads = (int)a.heads, p.g = (int)(a.heads / c.kv_heads);
    p.row_tiles = q.row_tiles, p.splits = q.splits, p.chunk = q.chunk;
    p.magic = kv8_magic((uint32_t)(c.page_size / kKv8Block));
    p.f = a.scale * 1.4426950408889634f;
    p.causal = a.causal, p.window = a.causal ? (int)a.window : 0;
    const int size = act_bytes(a.dtype);
    p.vec = (((uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)(a.q_token * size) | (uintptr_t)(a.out_token * size)) & 15u) == 0;
    p.count = static_cast<unsigned *>(a.workspace);
    p.part = reinterpret_cast<float *>(static_cast<char *>(a.workspace) + kWorkspaceCounterHead);
    p.stat = p.part + q.part_floats;
    const void *fn = a.dtype == VKQ_F32   ? decode_fn<float>(c.head_dim, p.pool.e4m3, q.rows)
                     : a.dtype == VKQ_F16 ? decode_fn<__half>(c.head_dim, p.pool.e4m3, q.rows)
                                          : decode_fn<__nv_bfloat16>(c.head_dim, p.pool.e4m3, q.rows);
    const size_t slots = (size_t)kDecWarps * kDecStages * (4 * kKv8Block * c.head_dim + 16);
    const size_t join = (size_t)kDecWarps * q.rows * (c.head_dim + 2) * sizeof(float);
    const size_t smem = slots > join ? slots : join;
    cudaError_t e = kernel_smem(fn, smem, true);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(q.splits * q.row_tiles), (unsigned)c.kv_heads, (unsigned)b.batch);
    cfg.blockDim = dim3(kDecThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    void *args[] = {(void *)&p};
    return cudaLaunchKernelExC(&cfg, fn, args);
}

int *kv8_attention_status_word() { return status_word(g_kv8_attn_status); }

}  // namespace vkq
