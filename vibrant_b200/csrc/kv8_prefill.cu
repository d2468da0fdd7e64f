// kv8_prefill.cu -- attention of many query rows (chunks of prompts) over the
// 8-bit paged KV cache, on tcgen05 with TMEM.
//
// The rows of a tile are (new token, query head) pairs of one sequence and KV
// head, as in kv8_attention.cu, so the heads of a group share every key tile.
// A CTA (one per SM, four warpgroups) takes one tile of rows and a range of
// keys in tiles of 128:
//   a warp of warpgroup 3 looks the tiles' pages up and copies their codes to
//     shared memory, 16 tokens of a head (1 or 2 KB) a bulk copy, a ring of three;
//   warpgroup 2 turns them into float16 K and V tiles (exact; 128-byte swizzle,
//     one layout read K-major as K and MN-major as V), a ring of three;
//   other warps of warpgroup 3 (one a half of the rows) issue the products;
//   warpgroups 0 and 1 work on the scores, a thread a row.
// The block scales never touch the operands.  With x = f ks (q . ck) the
// score of a key in units of log2 and lv = log2 vs,
//   e = exp2(x + lv - M),  M the running maximum of x + lv,
//   O = sum e cv,  l = sum e / vs,  o = O / l:
// vs goes into the exponent, so that the second product's operand stays
// within (0, 1], and out of the sum.  Both scales of 16 keys cost a thread two
// multiplications a tile.  The price: e ends, as a float16 operand, at 2^-39 of
// the row's largest p vs (float32) or 2^-31 (16-bit, whose M may be 2^8 behind),
// not of its largest p, so a dimension in which blocks of far larger scales
// hold zeros sees fewer digits of the others.  l comes from the float32 e.
//
// 16-bit q: 256 rows in two halves, each with a warpgroup, an issuing warp and
// two score buffers of 64 keys: the scores of the next 64 keys are computed
// while a warpgroup works on the ones before, and a K or V tile is converted
// once for 256 rows.  e is rounded to 11 bits; the output stays in TMEM, and M
// is raised (and the output rescaled) only when the maximum grew by more than
// 2^8, which the operand's range allows.
// float32 q: 128 rows; q and e are split into two 11-bit parts, so a tile
// takes the same four products, every key tile's output starts from zero, and
// warpgroup 1 adds it to float32 registers while warpgroup 0 works on the next
// scores.
//
// The matrix unit's accumulators round toward zero, and that adds up: values of
// one sign lose 6.2e-9 of their sum a key (measured: 4.1e-4 over 66,700 keys).
// That is why float32 adds tile by tile, and 16-bit q moves its output to
// float32 sums in the workspace every kMoveF16 or kMoveBf16 keys.
//
// Row tiles go from each sequence's last (which sees most keys) to its first, so
// that the longest start first.  Few tiles are split along the keys, and their parts
// added in order by kv8_join_kernel.
//
// The copies and the conversion start while q is still on its way; an output
// row goes out through shared memory, a whole line a store.  Loops that run
// once a key tile stay together in the source, and are not unrolled further
// than they need: with the start and the end of a block between them, their
// instructions no longer stayed in the caches (4,096 tokens: 687 instead of
// 620 us).
//
// Measured, 40 heads on 8 of D = 128: 4,096 new tokens of 8,192 in bfloat16 620
// us, 830 TFLOP/s of q K and e V (1,843 of 12,288: 446 us, 960), in float32,
// which takes four products for two, 1.10 ms; what bounds both is the hand-over
// from loads to conversion to products to scores: without it the tensor pipe
// would need 310 us, as it does twice that in float32.
#include <atomic>
#include <cmath>
#include <cstdint>

#include "../../include/vkq.h"
#include "act.cuh"
#include "kq_device.cuh"
#include "kv8.cuh"
#include "umma.cuh"
#include "vkq_internal.h"

namespace vkq {

static __device__ int g_kv8_prefill_status;

constexpr int kPreThreads = 512;
constexpr int kPreKeys = 128;                    // keys of a tile
constexpr int kPreBlocks = kPreKeys / kKv8Block;  // and its scale blocks
constexpr int kPreSub = 64;                       // keys whose scores a thread holds at once
constexpr int kPreRing = 3;  // float16 tiles
constexpr int kPreRaw = 3;   // tiles of codes
constexpr uint32_t kPrePolls = 1u << 27;
// Keys after which 16-bit q moves its output out of TMEM: 1.0e-4 and 4.1e-4 lost
// at most, a fifth and a tenth of the rounding of a float16 or bfloat16 output
// (half a unit, 2^-11 and 2^-8).  Measured, 4,096 float16 tokens of 200,000, 40
// heads on 8 of D = 128: 9.2e-5 lost and 20.8 ms, 4.1e-4 and 20.7 ms without;
// ranges of so many keys instead took 24.8 ms and five times the workspace.
constexpr int kMoveF16 = 16384, kMoveBf16 = 65536;
// and the score warps' passes that they are
template <typename T> constexpr int kMovePasses = kMoveF16 / kPreSub;
template <> constexpr int kMovePasses<__nv_bfloat16> = kMoveBf16 / kPreSub;
// registers a thread of warpgroups 0 and 1, of 2, of 3: at most 4 x 128 in all
// (float32: warpgroup 1 holds a row's output)
template <bool SPLIT> struct PreRegs {
    static constexpr int score = SPLIT ? 176 : 152, convert = SPLIT ? 72 : 96, issue = SPLIT ? 88 : 112;
    static_assert(2 * score + convert + issue <= 512, "more than the launch has");
    static_assert(score > 128 && convert < 128 && issue < 128, "setmaxnreg.inc grows, setmaxnreg.dec shrinks");
};

struct PrefillParams {
    Kv8Pool pool;
    Kv8Batch batch;
    const void *q;
    void *out;
    int64_t qt, ot;
    int heads, g, row_tiles, splits, chunk;
    float f;  // scale * log2(e)
    int causal, window;
    bool vec;
    float *part, *stat;
};

// Products issued by a whole warp, one lane of which (`one`) is the issuer: the
// descriptors then stay in uniform registers.  A shared-memory descriptor is
// given by its low word (address and leading offset) and its constant high one.
__device__ __forceinline__ void umma_f16(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, uint32_t acc,
                                         uint32_t one) {
    asm volatile(
        "{ .reg .pred p, q; .reg .b64 x, y; mov.b64 x, {%1, %3}; mov.b64 y, {%2, %3}; setp.ne.b32 p, %5, 0; "
        "setp.ne.b32 q, %6, 0; @q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %4, p; }" ::"r"(d),
        "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(acc), "r"(one));
}
// The first operand in TMEM: a row a lane, two float16 a column.
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, uint32_t acc,
                                            uint32_t one) {
    asm volatile(
        "{ .reg .pred p, q; .reg .b64 y; mov.b64 y, {%2, %3}; setp.ne.b32 p, %5, 0; setp.ne.b32 q, %6, 0; "
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p; }" ::"r"(d),
        "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(acc), "r"(one));
}
__device__ __forceinline__ void umma_commit_one(uint32_t bar, uint32_t one) {
    asm volatile(
        "{ .reg .pred q; setp.ne.b32 q, %1, 0; "
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(bar),
        "r"(one)
        : "memory");
}
__host__ __device__ constexpr uint32_t desc_hi(uint32_t sbo) { return (sbo >> 4) | (1u << 14) | (2u << 29); }
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return (addr >> 4) | ((lbo >> 4) << 16); }
// float16 operands, float32 accumulation, 128 rows; vn: the second operand N-major.
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool vn) {
    return (1u << 4) | ((vn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

// 32 consecutive TMEM columns of the thread's lane; the caller waits (tmem_wait_ld) before using them.
__device__ __forceinline__ void tmem_ld32(uint32_t (&r)[32], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
        "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
          "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
          "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {"
        "%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
        "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
// Waits for the thread's TMEM loads; r passes through, so that no use of it moves above the wait.
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                 "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                 "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 ::"memory");
}
// The same with eight and sixteen columns.
__device__ __forceinline__ void tmem_ld8(uint32_t (&r)[8], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]),
                   "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
                 ::"memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ float ex2p(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_half(uint32_t b) { return __half22float2(*reinterpret_cast<const __half2 *>(&b)); }
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// Polls a phase, kPrePolls times at most (some seconds): a small loop, because
// the roles' code has to stay in the instruction caches together.
__device__ __forceinline__ bool poll(uint32_t bar, uint32_t parity) {
#pragma unroll 1
    for (uint32_t i = 0; i < kPrePolls; i++)
        if (mbar_test_wait(bar, parity)) return true;
    return false;
}

// 16 codes as 16 float16.
template <bool E4M3>
__device__ __forceinline__ void codes_to_half(const uint4 &raw, uint32_t (&h)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t u = kv8_unsign<E4M3>(w[i]);
        h[2 * i] = kv8_widen<E4M3, false>(u);
        h[2 * i + 1] = kv8_widen<E4M3, true>(u);
    }
}

// Byte offset of 16-byte piece pc (of D / 8) of row r in a float16 tile of
// 128 rows: halves of 64 values, 128-byte rows, pieces swizzled by the row.
__device__ __forceinline__ uint32_t tile_off(int r, int pc) {
    return (uint32_t)((pc >> 3) * (kPreKeys * 128) + r * 128 + (((pc & 7) ^ (r & 7)) << 4));
}

// The keys that a tile of rows from r0 sees, and the ranges they are split into.
struct PreKeySpan {
    int lo, hi, active;
};
__device__ __forceinline__ PreKeySpan pre_keys(const PrefillParams &p, const Kv8Seq &s, int r0, int rows) {
    const int pos0 = s.len - s.n, row_end = min(r0 + rows, s.n * p.g) - 1;
    PreKeySpan k;
    k.hi = p.causal ? max(pos0 + row_end / p.g + 1, 0) : s.len;
    k.lo = 0;
    if (p.window > 0) k.lo = max(pos0 + r0 / p.g - p.window + 1, 0) & ~(kKv8Block - 1);
    k.active = max((k.hi - k.lo + p.chunk - 1) / p.chunk, 1);
    return k;
}

template <typename T, int D, bool E4M3>
__global__ void __launch_bounds__(kPreThreads, 1) kv8_prefill_kernel(const PrefillParams p) {
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int ROWS = SPLIT ? 128 : 256;
    constexpr uint32_t TILE = 128 * D * 2;          // bytes of a float16 tile of 128 rows
    constexpr uint32_t HALF = kPreKeys * 128;       // its second half of 64 values
    constexpr float kUp = SPLIT ? 14.f : 6.f;       // e is held as 2^kUp e (at most 2^14)
    // TMEM columns: the scores (and, over them, e) of half or parity 0 and 1, the outputs
    constexpr uint32_t kS = 0, kO = 256;
    extern __shared__ __align__(1024) uint8_t smem[];  // two q tiles, the rings
    __shared__ __align__(8) uint64_t bars[2 * kPreRing + 2 * kPreRaw + 4 + 4 + 2 + 2 + 1];
    __shared__ __align__(16) float scales[8][3][kPreBlocks];  // of key tile j & 7: ks, lv, 1 / vs
    __shared__ float alpha[4][128], lsum[128], msum[128], row_f[ROWS];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t abort_flag;
    __shared__ uint32_t bad_flag;
    __shared__ int64_t q_row[ROWS], out_row[ROWS];  // where the rows are (out: -1 past the last)
    pdl_wait();
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = warp >> 2, t = tid & 127;
    // block = ((reversed row tile, range), sequence, KV head), the last fastest
    const int kvh = (int)(blockIdx.x % p.pool.kv_heads), x0 = (int)(blockIdx.x / p.pool.kv_heads);
    const int seq = x0 % (int)p.batch.batch, x1 = x0 / (int)p.batch.batch;
    const int split = x1 % p.splits;
    const Kv8Seq s = kv8_seq(p.batch, p.pool.page, seq);
    const int rows_all = s.n * p.g;
    const int rt = (rows_all + ROWS - 1) / ROWS - 1 - x1 / p.splits;  // from the sequence's own last
    const int r0 = rt * ROWS;
    if (!s.ok) {
        if (split > 0) return;
        if (tid == 0) atomicExch(&g_kv8_prefill_status, VKQ_ERR_INVALID_ARGUMENT);
        if (rt < 0) return;
        for (int64_t i = tid; i < (int64_t)ROWS * D; i += kPreThreads) {
            const int r = r0 + (int)(i / D);
            if (r < rows_all)
                static_cast<T *>(p.out)[(int64_t)(s.first + r / p.g) * p.ot + (int64_t)(kvh * p.g + r % p.g) * D + i % D] =
                    from_f32<T>(__int_as_float(0x7fc00000));
        }
        return;
    }
    if (rt < 0) return;
    const int pos0 = s.len - s.n;
    const PreKeySpan span = pre_keys(p, s, r0, ROWS);
    const int lo = span.lo, hi = span.hi, active = span.active;
    if (split >= active) return;
    const int k_lo = lo + split * p.chunk, k_hi = min(hi, k_lo + p.chunk);
    const int n = k_hi > k_lo ? (k_hi - k_lo + kPreKeys - 1) / kPreKeys : 0;  // key tiles
    const bool two = !SPLIT && rows_all - r0 > 128;  // the second half has rows

    const uint32_t base = (smem_u32addr(smem) + 1023u) & ~1023u;
    const uint32_t q_tile = base, ring = base + 2 * TILE, raw = ring + kPreRing * TILE;
    auto bar = [&](int i) { return smem_u32addr(&bars[i]); };
    constexpr int FULL = 0, EMPTY = kPreRing, RF = 2 * kPreRing, RE = RF + kPreRaw, SF = RE + kPreRaw, PF = SF + 4, TF = PF + 4,
                  TE = TF + 2, DR = TE + 2;
    if (tid == 0) {
        for (int i = 0; i < kPreRing; i++) {
            mbar_init(bar(FULL + i), 4);   // a lane of each converting warp
            mbar_init(bar(EMPTY + i), two ? 2 : 1);  // commits
        }
        for (int i = 0; i < kPreRaw; i++) {
            mbar_init(bar(RF + i), 1);  // the copies' bytes
            mbar_init(bar(RE + i), 4);  // a lane of each converting warp
        }
        for (int i = 0; i < 4; i++) {  // of a half's two score buffers (SPLIT: of the two)
            mbar_init(bar(SF + i), 1);  // commit: scores
            mbar_init(bar(PF + i), 4);  // e is in TMEM
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(bar(TF + i), 1);              // commit: a half's output (SPLIT: of one key tile)
            mbar_init(bar(TE + i), SPLIT ? 4 : 1);  // commit: a half's output up to a tile (SPLIT: it has been read)
        }
        mbar_init(bar(DR), two ? 2 : 1);  // commits: an issuer's last
        mbar_init_fence();
        abort_flag = 0;
        bad_flag = 0;
    }
    __syncthreads();
    uint32_t tmem = 0;
    // The copies and the conversion start at once; those who need q and TMEM
    // (warpgroups 0 and 1, the issuing warps) meet here.
    auto meet = [&]() {
        fence_before();
        asm volatile("bar.sync 2, 320;" ::: "memory");
        fence_after();
        tmem = tmem_slot;
    };

    // for whole warps: one lane polls
    auto wait_warp = [&](uint32_t b, uint32_t parity) -> bool {
        int ok = 1;
        if (lane == 0 && !poll(b, parity)) ok = 0, abort_flag = 1;
        return __shfl_sync(0xffffffffu, ok, 0) != 0;
    };
    auto arrive = [&](uint32_t b) {  // once for the warp, after all its lanes
        __syncwarp();
        if (lane == 0) mbar_arrive(b);
    };

    const int64_t tile = ((int64_t)seq * p.pool.kv_heads + kvh) * p.row_tiles + rt;
    const float nan = __int_as_float(0x7fc00000);
    const int row = SPLIT ? t : 128 * wg + t;  // of warpgroups 0 and 1
    int row_token = 0;
    bool there = false;
    float m = -INFINITY, l = 0.f;
    float moved_m = -INFINITY;  // the M of what the row's output has moved to the workspace
    // the row's sums there, four dimensions at ROWS float4 a step (16-bit q, and the parts of ranges)
    auto moved = [&]() { return reinterpret_cast<float4 *>(p.part + (tile * p.splits + split) * ROWS * D) + row; };
    auto add_moved = [&](float (&x)[8], const float4 *d, float k) {
        const float4 a = d[0], b = d[ROWS];
        x[0] = fmaf(a.x, k, x[0]), x[1] = fmaf(a.y, k, x[1]), x[2] = fmaf(a.z, k, x[2]), x[3] = fmaf(a.w, k, x[3]);
        x[4] = fmaf(b.x, k, x[4]), x[5] = fmaf(b.y, k, x[5]), x[6] = fmaf(b.z, k, x[6]), x[7] = fmaf(b.w, k, x[7]);
    };
    if (wg < 2) {
        there = r0 + row < rows_all;
        row_token = there ? (r0 + row) / p.g : 0;
        const int row_head = kvh * p.g + (there ? r0 + row - row_token * p.g : 0);
        if (!SPLIT || wg == 0) {
            q_row[row] = (int64_t)(s.first + row_token) * p.qt + (int64_t)row_head * D;
            out_row[row] = there ? (int64_t)(s.first + row_token) * p.ot + (int64_t)row_head * D : -1;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        // q: consecutive lanes load a row's consecutive eight values, scale them
        // by the row's power of two, below 2^15, and store the float16 tile
        // (SPLIT: both parts)
        {
            constexpr int PR = D / 8, PIECES = ROWS * PR / 256, QB = SPLIT || PIECES < 8 ? 4 : 8;
#pragma unroll 1
            for (int b0 = 0; b0 < PIECES; b0 += QB) {
                float x[QB][8];
#pragma unroll
                for (int b = 0; b < QB; b++) {
                    const int lr = ((b0 + b) * 256 + tid) / PR;
                    load_act<T, 8>(static_cast<const T *>(p.q) + q_row[lr] + tid % PR * 8, x[b], p.vec);
                }
#pragma unroll
                for (int b = 0; b < QB; b++) {
                    const int lr = ((b0 + b) * 256 + tid) / PR;
                    float a = 0.f;
#pragma unroll
                    for (int u = 0; u < 8; u++) a = fmaxf(a, fabsf(x[b][u]));
#pragma unroll
                    for (int o = 1; o < PR; o <<= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
                    const int e = min(max((int)(__float_as_uint(a) >> 23) - 127, -60), 127);
                    const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23);
                    if (tid % PR == 0) row_f[lr] = p.f * __uint_as_float((uint32_t)(e - 14 + 127) << 23);
                    const uint32_t dst = q_tile + (SPLIT ? 0u : (uint32_t)(lr / 128) * TILE) + tile_off(lr % 128, tid % PR);
                    uint32_t w[4], w2[4];
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const float x0 = x[b][2 * u] * up, x1 = x[b][2 * u + 1] * up;
                        w[u] = pack_half(x0, x1);
                        if constexpr (SPLIT) {
                            const float2 back = unpack_half(w[u]);
                            w2[u] = pack_half(x0 - back.x, x1 - back.y);
                        }
                    }
                    sts128(dst, w[0], w[1], w[2], w[3]);
                    if constexpr (SPLIT) sts128(dst + TILE, w2[0], w2[1], w2[2], w2[3]);
                }
            }
            fence_async();
            meet();
        }
    }
    // The tiles in the order in which the products take them: K0, then V(j),
    // K(j + 1) (SPLIT: K(j + 1), V(j): the scores of a tile are asked for before
    // the output of the one before).
    struct Item {
        int j, k_done, v_done;  // key tile; K and V tiles up to and with this one
        bool is_v;
    };
    auto after = [&](const Item &a) {
        Item b;
        b.is_v = SPLIT ? !(a.k_done < n && a.k_done < a.v_done + 2) : a.v_done < a.k_done;
        b.j = b.is_v ? a.v_done : a.k_done;
        b.k_done = a.k_done + !b.is_v, b.v_done = a.v_done + b.is_v;
        return b;
    };
            // Eight values from dimension c.  A row of out goes through shared memory
            // (the half's q tile, done with by then), in pieces of 16 bytes swizzled
            // by the row, so that a warp stores whole lines: rows stored by their
            // threads took 8,000 clocks a block.
            // (What they need is worked out here: kept over the loop it cost registers
            // there, and 3% of a long prompt's time.)
            constexpr int PC = D * (int)sizeof(T) / 16, N = 16 / (int)sizeof(T);
            auto stage = [&]() { return smem + (q_tile - smem_u32addr(smem)) + (SPLIT ? 0u : wg * TILE); };
            auto put = [&](int c, float (&v)[8], float inv) {
                if (active > 1) {  // this range's part, rows fastest
                    float *const part = p.part + (tile * p.splits + split) * ROWS * D;
                float4 *d = reinterpret_cast<float4 *>(part) + c / 4 * ROWS + row;
                    d[0] = make_float4(v[0], v[1], v[2], v[3]);
                    d[ROWS] = make_float4(v[4], v[5], v[6], v[7]);
                } else {
    #pragma unroll
                    for (int u = 0; u < 8; u++) v[u] *= inv;
    #pragma unroll
                    for (int z = 0; z < 8; z += N) {
                        float piece[N];
    #pragma unroll
                        for (int u = 0; u < N; u++) piece[u] = v[z + u];
                        store_act<T, N>(reinterpret_cast<T *>(stage() + t * (16 * PC) + ((((c + z) / N) ^ (t & 7)) << 4)), piece, true);
                    }
                }
            };
            auto put_stat = [&](float m, float l) {
                if (active > 1) reinterpret_cast<float2 *>(p.stat + (tile * p.splits + split) * ROWS * 2)[row] = make_float2(m, l);
            };
            auto put_end = [&]() {
                if (active > 1) return;
                __syncwarp();
    #pragma unroll 4
                for (int i = lane; i < 32 * PC; i += 32) {
                    const int from = 32 * (warp & 3) + i / PC, pc = i % PC;
                    const int64_t o = out_row[SPLIT ? from : 128 * wg + from];
                    if (o < 0) continue;
                    const uint4 v = *reinterpret_cast<const uint4 *>(stage() + from * (16 * PC) + ((pc ^ (from & 7)) << 4));
                    T *const dst = static_cast<T *>(p.out) + o + pc * N;
                    if (p.vec) {
                        *reinterpret_cast<uint4 *>(dst) = v;
                    } else {
                        alignas(16) T e[N];
                        *reinterpret_cast<uint4 *>(e) = v;
    #pragma unroll
                        for (int u = 0; u < N; u++) dst[u] = e[u];
                    }
                }
            };
    if (wg == 2) {
        // ---- codes to float16 tiles ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PreRegs<SPLIT>::convert));
        // A thread takes 16-byte pieces: piece ch of rows row0, row0 + RSTEP, ...
        // Eight lanes that store together hold two rows of unlike parity and four
        // pieces of one half, which the swizzle puts into different banks.
        constexpr int PER = kPreKeys * D / 16 / 128;  // 8 (D = 128) or 4
        constexpr int RSTEP = kPreKeys / PER;         // 16 or 32
        const int row0 = D == 128 ? 4 * (warp & 3) + (lane >> 4) * 2 + ((lane >> 2) & 1) : t / 4;
        const int ch = D == 128 ? (lane & 3) + 4 * ((lane >> 3) & 1) : t % 4;
        const uint32_t st0 = tile_off(row0, 2 * ch), st1 = tile_off(row0, 2 * ch + 1);  // RSTEP rows: RSTEP * 128 bytes
        Item item{0, 1, 0, false};
        RingPos rp, rr;
        for (int it = 0; it < 2 * n; it++) {
            if (!wait_warp(bar(RF + rr.idx), rr.phase)) break;
            if (rp.uses >= (uint32_t)kPreRing && !wait_warp(bar(EMPTY + rp.idx), rp.phase ^ 1u)) break;
            const uint32_t dst = ring + rp.idx * TILE, src = raw + rr.idx * (TILE / 2) + (uint32_t)(row0 * D + ch * 16);
            const int left = k_hi - (k_lo + item.j * kPreKeys) - row0;  // rows past the range are zeros
#pragma unroll 1
            for (int k = 0; k < PER; k++) {
                uint4 c = lds128(src + (uint32_t)k * (RSTEP * D));
                if (k * RSTEP >= left) c = make_uint4(0, 0, 0, 0);
                uint32_t h[8];
                codes_to_half<E4M3>(c, h);
                sts128(dst + st0 + (uint32_t)k * (RSTEP * 128), h[0], h[1], h[2], h[3]);
                sts128(dst + st1 + (uint32_t)k * (RSTEP * 128), h[4], h[5], h[6], h[7]);
            }
            fence_async();
            arrive(bar(FULL + rp.idx));
            if (lane == 0) mbar_arrive(bar(RE + rr.idx));
            rp.next(kPreRing);
            rr.next(kPreRaw);
            item = after(item);
        }
    } else if (wg == 3) {
        // ---- the products ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PreRegs<SPLIT>::issue));
        if (warp == 12) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32addr(&tmem_slot)));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
        if (warp == 12 || warp == 14) meet();
        if (warp == 13 && n > 0) {
            // the tiles' pages: lane b takes block b
            const uint32_t per_page = (uint32_t)(p.pool.page / kKv8Block), magic = 0xffffffffu / per_page + 1u;
            // The block of the layer's pool ([page][kv head][block]): 0 past the range
            // and, with bad_flag, for a page out of range.  (Below 2^31: a pool of
            // that many blocks would be 2 TB.)
            auto look = [&](int j) -> uint32_t {
                const int key = k_lo + j * kPreKeys + lane * kKv8Block;
                if (lane >= kPreBlocks || j >= n || key >= k_hi) return 0;
                const uint32_t blk = (uint32_t)key / kKv8Block, lp = kv8_div(blk, per_page, magic);
                const int id = kv8_page(p.pool, s, (int)lp);
                if (id < 0) bad_flag = 1;
                return id < 0 ? 0u : ((uint32_t)id * (uint32_t)p.pool.kv_heads + (uint32_t)kvh) * per_page + (blk - lp * per_page);
            };
            Item item{0, 1, 0, false};
            uint32_t at = look(0);
            RingPos rr;
            for (int it = 0; it < 2 * n; it++) {
                const Item next = after(item);
                const uint32_t at_next = look(next.j);  // looked up while this tile's slot is waited for
                const int left = k_hi - (k_lo + item.j * kPreKeys);
                const int blocks = min((left + kKv8Block - 1) / kKv8Block, kPreBlocks);
                float ks = 1.f, vs = 1.f;
                if (!item.is_v && lane < blocks) ks = p.pool.ks[at], vs = p.pool.vs[at];
                if (rr.uses >= (uint32_t)kPreRaw && !wait_warp(bar(RE + rr.idx), rr.phase ^ 1u)) break;
                if (!item.is_v && lane < kPreBlocks) {
                    scales[item.j & 7][0][lane] = ks;
                    scales[item.j & 7][1][lane] = __log2f(vs);
                    scales[item.j & 7][2][lane] = 1.f / vs;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive_expect_tx(bar(RF + rr.idx), (uint32_t)blocks * (kKv8Block * D));
                __syncwarp();
                if (lane < blocks)
                    bulk_g2s(raw + rr.idx * (TILE / 2) + (uint32_t)lane * (kKv8Block * D),
                             (item.is_v ? p.pool.v : p.pool.k) + (uint64_t)at * (kKv8Block * D), kKv8Block * D,
                             bar(RF + rr.idx));
                rr.next(kPreRaw);
                item = next;
                at = at_next;
            }
            // every copy has landed before the block ends
            if (lane == 0)
                for (uint32_t i = 0; i < (uint32_t)kPreRaw; i++) {
                    const uint32_t uses = rr.uses / kPreRaw + (i < rr.uses % kPreRaw ? 1u : 0u);
                    if (uses) poll(bar(RF + i), (uses - 1) & 1u);
                }
            __syncwarp();
        } else if ((warp == 12 || (warp == 14 && two)) && n > 0) {
            // one issuer; with two halves one each (they share no scores or output)
            constexpr uint32_t IQK = idesc_f16(SPLIT ? kPreKeys : kPreSub, false), IPV = idesc_f16(D, true);
            constexpr uint32_t HI = desc_hi(1024);  // eight rows of 128 bytes
            const uint32_t one = lane == 0;
            RingPos rp;
            bool ok = true;
            auto take = [&](uint32_t &slot) {
                slot = rp.idx;
                ok = ok && wait_warp(bar(FULL + rp.idx), rp.phase);
                fence_after();
                rp.next(kPreRing);
            };
            // scores = q tile x K; K-major both: 16 values are 32 bytes into a 128-byte row
            auto qk = [&](uint32_t d, uint32_t q, uint32_t k_tile, bool acc) {
                const uint32_t da = desc_lo(q, 16u), db = desc_lo(k_tile, 16u);
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    const uint32_t off = ((k >> 2) * HALF + (k & 3) * 32u) >> 4;
                    umma_f16(d, da + off, db + off, HI, IQK, (k > 0 || acc) ? 1u : 0u, one);
                }
            };
            // output = e x V; e: 16 keys are 8 of every 32 columns' first 16; V N-major: 16 keys
            // are 2048 bytes, the next 64 values HALF further
            auto pv = [&](uint32_t d, uint32_t e, uint32_t v_tile, bool acc) {
                const uint32_t db = desc_lo(v_tile, HALF);
#pragma unroll
                for (int k = 0; k < (SPLIT ? kPreKeys : kPreSub) / 16; k++)
                    umma_f16_ts(d, e + 32u * (k >> 1) + 8u * (k & 1), db + (k * 2048u >> 4), HI, IPV,
                                (k > 0 || acc) ? 1u : 0u, one);
            };
            auto commit = [&](uint32_t b) { umma_commit_one(b, one); };
            uint32_t ks, vs;
            if constexpr (SPLIT) {
                auto scores = [&](int j) {
                    take(ks);
                    if (!ok) return;
                    const uint32_t d = tmem + kS + 128u * (j & 1);
                    qk(d, q_tile, ring + ks * TILE, false);
                    qk(d, q_tile + TILE, ring + ks * TILE, true);
                    commit(bar(SF + (j & 1)));
                    commit(bar(EMPTY + ks));
                };
                scores(0);
                if (ok && n > 1) scores(1);
                for (int j = 0; j < n && ok; j++) {
                    const uint32_t b = j & 1, ph = (j >> 1) & 1;
                    take(vs);
                    if (ok && j >= 2) ok = wait_warp(bar(TE + b), ph ^ 1u);
                    if (ok) ok = wait_warp(bar(PF + b), ph);
                    if (!ok) break;
                    fence_after();
                    const uint32_t d = tmem + kO + 128u * b, e = tmem + kS + 128u * b;
                    pv(d, e, ring + vs * TILE, false);
                    pv(d, e + 16u, ring + vs * TILE, true);
                    commit(bar(TF + b));
                    commit(bar(EMPTY + vs));
                    if (j + 2 < n) scores(j + 2);
                }
            } else {
                const uint32_t hf = warp == 14, sc = tmem + kS + 128u * hf, o = tmem + kO + 128u * hf;
                const uint32_t sf = SF + 2 * hf, pf = PF + 2 * hf;
                // 64 keys of a tile are 8 KB of each half of its values
                auto scores = [&](uint32_t b) {
                    qk(sc + (uint32_t)kPreSub * b, q_tile + hf * TILE, ring + ks * TILE + b * (kPreSub * 128u), false);
                    commit(bar(sf + b));
                    if (b) commit(bar(EMPTY + ks));
                };
                take(ks);
                if (ok) scores(0), scores(1);
                for (int i = 0; i < 2 * n && ok; i++) {
                    const uint32_t b = i & 1;
                    if (b == 0) take(vs);
                    ok = ok && wait_warp(bar(pf + b), (i >> 1) & 1);
                    if (!ok) break;
                    fence_after();
                    pv(o, sc + kPreSub * b, ring + vs * TILE + b * (kPreSub * 128u), i > 0);
                    commit(bar(TE + hf));
                    if (b) commit(bar(EMPTY + vs));
                    if (i + 2 < 2 * n) {
                        if (b == 0) take(ks);
                        if (!ok) break;
                        scores(b);
                    }
                }
                commit(bar(TF + hf));
            }
            // every product issued has finished before TMEM is given back
            commit(bar(DR));
            if (warp == 12) wait_warp(bar(DR), 0);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PreRegs<SPLIT>::score));
        const uint32_t my = tmem + ((uint32_t)(32 * (warp & 3)) << 16);  // the warp's lanes
        if (wg == 0 || (!SPLIT && two)) {
            // ---- scores to e ----
            const int ps = pos0 + row_token;  // the row's position; it sees [see_lo, see_hi)
            const int see_hi = !there ? 0 : min(p.causal ? ps + 1 : s.len, k_hi);
            const int see_lo = p.window > 0 ? ps - p.window + 1 : 0;
            const float rf = row_f[row];
            const int warp_hi = __reduce_min_sync(0xffffffffu, see_hi), warp_lo = __reduce_max_sync(0xffffffffu, see_lo);
            bool ok = true;
            // a pass: 64 keys (SPLIT: a tile, its 64 scores at a time read twice)
            constexpr int PARTS = SPLIT ? kPreKeys / kPreSub : 1;
            const uint32_t hf = SPLIT ? 0 : wg;
            for (int i = 0; i < (SPLIT ? n : 2 * n) && ok; i++) {
                const uint32_t b = i & 1, ph = (i >> 1) & 1;
                ok = wait_warp(bar(SF + 2 * hf + b), ph);
                if (!ok) break;
                fence_after();
                const uint32_t sc = my + kS + (SPLIT ? 128u * b : 128u * hf + kPreSub * b);
                const int j = SPLIT ? i : i >> 1;
                const float *scl = scales[j & 7][0] + (SPLIT ? 0 : 4 * b);  // ks; lv and 1 / vs kPreBlocks further each
                const int key = k_lo + i * (SPLIT ? kPreKeys : kPreSub);
                const bool edge = key < warp_lo || key + (SPLIT ? kPreKeys : kPreSub) > warp_hi;
                uint32_t x[2][32];
                float kf[4], lv[4];
                auto load = [&](int h) {
                    tmem_ld32(x[0], sc + kPreSub * h);
                    tmem_ld32(x[1], sc + kPreSub * h + 32u);
                    const float4 a = *reinterpret_cast<const float4 *>(scl + 4 * h);
                    const float4 c = *reinterpret_cast<const float4 *>(scl + kPreBlocks + 4 * h);
                    // the factor above 0: -inf stays -inf
                    kf[0] = fmaxf(a.x * rf, 1.4e-45f), kf[1] = fmaxf(a.y * rf, 1.4e-45f);
                    kf[2] = fmaxf(a.z * rf, 1.4e-45f), kf[3] = fmaxf(a.w * rf, 1.4e-45f);
                    lv[0] = c.x, lv[1] = c.y, lv[2] = c.z, lv[3] = c.w;
                    tmem_wait_ld(x[0]);
                    tmem_wait_ld(x[1]);
                    if (edge) {
                        const int k0 = see_lo - key - kPreSub * h, k1 = see_hi - key - kPreSub * h;  // visible: [k0, k1)
#pragma unroll
                        for (int u = 0; u < kPreSub; u++)
                            if (u < k0 || u >= k1) x[u / 32][u % 32] = 0xff800000u;  // -inf
                    }
                };
                // the maximum of x + lv
                float mx = m;
#pragma unroll 1
                for (int h = 0; h < PARTS; h++) {
                    load(h);
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const uint32_t *y = x[q / 2] + 16 * (q % 2);
                        float a[4];
#pragma unroll
                        for (int u = 0; u < 4; u++)  // short chains: four at a time
                            a[u] = fmaxf(fmaxf(__uint_as_float(y[4 * u]), __uint_as_float(y[4 * u + 1])),
                                         fmaxf(__uint_as_float(y[4 * u + 2]), __uint_as_float(y[4 * u + 3])));
                        mx = fmaxf(mx, fmaf(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])), kf[q], lv[q]));
                    }
                }
                float al = 1.f;
                if constexpr (SPLIT) {
                    al = mx == -INFINITY ? 1.f : ex2p(m - mx);
                    alpha[j & 3][t] = al;
                    m = mx;
                } else {
                    // raised only when e would pass 2^8: the output stays as it is otherwise
                    const bool raise = mx > m + 8.f;
                    const bool move = i > 0 && i % kMovePasses<T> == 0;
                    if (move || __any_sync(0xffffffffu, raise)) {
                        if (raise) {
                            al = ex2p(m - mx);
                            m = mx;
                        }
                        if (i > 0) {
                            ok = wait_warp(bar(TE + hf), (i - 1) & 1);  // the output of the keys before
                            if (!ok) break;
                            fence_after();
                            const uint32_t o0 = my + kO + 128u * hf;
                            if (!move) {
#pragma unroll 1
                                for (int c = 0; c < D / 8; c++) {
                                    uint32_t o[8];
                                    tmem_ld8(o, o0 + 8u * c);
                                    tmem_wait_ld(o);
#pragma unroll
                                    for (int u = 0; u < 8; u++) o[u] = __float_as_uint(__uint_as_float(o[u]) * al);
                                    tmem_st8(o0 + 8u * c, o);
                                }
                            } else {
                                const float old = moved_m == m ? 1.f : ex2p(moved_m - m);
                                moved_m = m;
                                float4 *d = moved();
#pragma unroll 1
                                for (int c = 0; c < D / 8; c++, d += 2 * ROWS) {
                                    uint32_t o[8];
                                    tmem_ld8(o, o0 + 8u * c);
                                    tmem_wait_ld(o);
                                    float x[8];
#pragma unroll
                                    for (int u = 0; u < 8; u++) x[u] = __uint_as_float(o[u]) * al, o[u] = 0u;
                                    if (i > kMovePasses<T>) add_moved(x, d, old);
                                    d[0] = make_float4(x[0], x[1], x[2], x[3]), d[ROWS] = make_float4(x[4], x[5], x[6], x[7]);
                                    tmem_st8(o0 + 8u * c, o);
                                }
                            }
                        }
                    }
                }
                l *= al;
                const float off = m == -INFINITY ? 0.f : m - kUp;
#pragma unroll 1
                for (int h = 0; h < PARTS; h++) {
                    if (PARTS > 1) load(h);
                    const float4 inv4 = *reinterpret_cast<const float4 *>(scl + 2 * kPreBlocks + 4 * h);
                    const float inv[4] = {inv4.x, inv4.y, inv4.z, inv4.w};
#pragma unroll
                    for (int q = 0; q < 2; q++) {  // 32 scores
                        uint32_t hp[16];
#pragma unroll
                        for (int z = 0; z < 2; z++) {
                            const float d = lv[2 * q + z] - off;
                            const float2 kf2 = make_float2(kf[2 * q + z], kf[2 * q + z]), d2 = make_float2(d, d);
                            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                            for (int u = 0; u < 8; u++) {
                                uint32_t *y = x[q] + 16 * z + 2 * u;
                                float2 e = f2fma(make_float2(__uint_as_float(y[0]), __uint_as_float(y[1])), kf2, d2);
                                e.x = ex2p(e.x), e.y = ex2p(e.y);
                                sum[u & 1] = f2add(sum[u & 1], e);
                                y[0] = __float_as_uint(e.x), y[1] = __float_as_uint(e.y);
                                hp[8 * z + u] = pack_half(e.x, e.y);
                            }
                            sum[0] = f2add(sum[0], sum[1]);
                            l = fmaf(sum[0].x + sum[0].y, inv[2 * q + z], l);
                        }
                        // e as float16 over its scores: 16 columns (SPLIT: the low parts in the 16 after)
                        tmem_st16(sc + kPreSub * h + 32u * q, hp);
                        if constexpr (SPLIT) {
#pragma unroll
                            for (int u = 0; u < 16; u++) {
                                const float2 back = unpack_half(hp[u]);
                                hp[u] = pack_half(__uint_as_float(x[q][2 * u]) - back.x, __uint_as_float(x[q][2 * u + 1]) - back.y);
                            }
                            tmem_st16(sc + kPreSub * h + 32u * q + 16u, hp);
                        }
                    }
                }
                tmem_wait_st();
                fence_before();
                arrive(bar(PF + 2 * hf + b));
            }
            if constexpr (SPLIT) {
                lsum[t] = l, msum[t] = m;
                asm volatile("bar.sync 1, 256;" ::: "memory");
            }
        } else if constexpr (SPLIT) {
            // ---- the key tiles' outputs, added in float32 ----
            float acc[D];
#pragma unroll
            for (int i = 0; i < D; i++) acc[i] = 0.f;
            for (int j = 0; j < n; j++) {
                const uint32_t b = j & 1;
                if (!wait_warp(bar(TF + b), (j >> 1) & 1)) break;
                fence_after();
                const float al = alpha[j & 3][t];
#pragma unroll
                for (int i = 0; i < D / 32; i++) {
                    uint32_t o[32];
                    tmem_ld32(o, my + kO + 128u * b + 32u * i);
                    tmem_wait_ld(o);
#pragma unroll
                    for (int u = 0; u < 32; u++) acc[32 * i + u] = fmaf(acc[32 * i + u], al, __uint_as_float(o[u]));
                }
                fence_before();
                arrive(bar(TE + b));
            }
            // l and M are warpgroup 0's: its last e came before the last output
            asm volatile("bar.sync 1, 256;" ::: "memory");
            l = lsum[t];
            if (bad_flag || abort_flag) l = nan;
            put_stat(msum[t], l);
            const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
            for (int c = 0; c < D; c += 8) {
                float v[8];
#pragma unroll
                for (int u = 0; u < 8; u++) v[u] = acc[c + u];
                put(c, v, inv);
            }
            put_end();
        }
    }
    if constexpr (!SPLIT) {
        if (wg == 0 || (wg == 1 && two)) {
            const bool got = n > 0 && wait_warp(bar(TF + wg), 0);
            fence_after();
            if (bad_flag || abort_flag) l = nan;
            put_stat(m, l);
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const bool add = 2 * n > kMovePasses<T>;
            const float old = moved_m == m ? 1.f : ex2p(moved_m - m);
#pragma unroll 1
            for (int i = 0; i < D / 32; i++) {
                uint32_t o[32];
                if (got) {
                    tmem_ld32(o, tmem + ((uint32_t)(32 * (warp & 3)) << 16) + kO + 128u * wg + 32u * i);
                    tmem_wait_ld(o);
                } else {
#pragma unroll
                    for (int u = 0; u < 32; u++) o[u] = 0;
                }
#pragma unroll
                for (int c = 0; c < 32; c += 8) {
                    float v[8];
#pragma unroll
                    for (int u = 0; u < 8; u++) v[u] = __uint_as_float(o[c + u]);
                    if (add) add_moved(v, moved() + (32 * i + c) / 4 * ROWS, old);
                    put(32 * i + c, v, inv);
                }
            }
            put_end();
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 12) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
    if (tid == 0) {
        if (bad_flag) atomicExch(&g_kv8_prefill_status, VKQ_ERR_INVALID_ARGUMENT);
        if (abort_flag) atomicExch(&g_kv8_prefill_status, kStatusTimeout);
    }
}

// The outputs of tiles that were split along the keys, the ranges' parts added
// in their order.  A block takes 32 rows, a warp an eighth of their values, a
// lane a row.  A launch of its own, because the last block of a tile to finish
// reads its ranges at one SM's bandwidth only: 12 us for 6 ranges of 256 rows.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv8_join_kernel(const PrefillParams p) {
    constexpr int ROWS = sizeof(T) == 4 ? 128 : 256, TD = D / 8, AT = 4;
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, d0 = (threadIdx.x >> 5) * TD;
    const int64_t tile = blockIdx.x / (ROWS / 32);
    const int rt = (int)(tile % p.row_tiles), kvh = (int)(tile / p.row_tiles % p.pool.kv_heads);
    const Kv8Seq s = kv8_seq(p.batch, p.pool.page, (int)(tile / p.row_tiles / p.pool.kv_heads));
    const int tr = (int)(blockIdx.x % (ROWS / 32)) * 32 + lane, r = rt * ROWS + tr;
    if (!s.ok || r >= s.n * p.g) return;
    const int active = pre_keys(p, s, rt * ROWS, ROWS).active;
    if (active < 2) return;
    const float4 *part = reinterpret_cast<const float4 *>(p.part + tile * p.splits * ROWS * D) + d0 / 4 * ROWS + tr;
    const float2 *stat = reinterpret_cast<const float2 *>(p.stat + tile * p.splits * ROWS * 2) + tr;
    float mx = -INFINITY, sum = 0.f, acc[TD];
#pragma unroll 8
    for (int w = 0; w < active; w++) mx = fmaxf(mx, __ldcg(stat + w * ROWS).x);
#pragma unroll
    for (int u = 0; u < TD; u++) acc[u] = 0.f;
    for (int w = 0; w < active; w += AT) {
        float4 v[AT][TD / 4];
        float2 ms[AT];
#pragma unroll
        for (int z = 0; z < AT; z++) {
            const bool is = w + z < active;
            ms[z] = is ? __ldcg(stat + (w + z) * ROWS) : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int u = 0; u < TD / 4; u++)
                v[z][u] = is ? __ldcg(part + (int64_t)(w + z) * (ROWS * D / 4) + u * ROWS) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int z = 0; z < AT; z++) {
            // a range without a visible key weighs nothing; a NaN sum spreads
            const float k = ms[z].x == -INFINITY ? (ms[z].y == ms[z].y ? 0.f : ms[z].y) : ex2p(ms[z].x - mx);
            sum = fmaf(k, ms[z].y, sum);
#pragma unroll
            for (int u = 0; u < TD / 4; u++) {
                acc[4 * u] = fmaf(k, v[z][u].x, acc[4 * u]), acc[4 * u + 1] = fmaf(k, v[z][u].y, acc[4 * u + 1]);
                acc[4 * u + 2] = fmaf(k, v[z][u].z, acc[4 * u + 2]), acc[4 * u + 3] = fmaf(k, v[z][u].w, acc[4 * u + 3]);
            }
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int u = 0; u < TD; u++) acc[u] *= inv;
    store_act<T, TD>(static_cast<T *>(p.out) + (int64_t)(s.first + r / p.g) * p.ot + (int64_t)(kvh * p.g + r % p.g) * D + d0, acc,
                     p.vec);
}

template <typename T, int D>
static const void *prefill_fn(bool e4m3) {
    return e4m3 ? (const void *)kv8_prefill_kernel<T, D, true> : (const void *)kv8_prefill_kernel<T, D, false>;
}
template <typename T>
static const void *prefill_fn(int D, bool e4m3) {
    return D == 64 ? prefill_fn<T, 64>(e4m3) : prefill_fn<T, 128>(e4m3);
}

template <typename T>
static const void *join_fn(int D) {
    return D == 64 ? (const void *)kv8_join_kernel<T, 64> : (const void *)kv8_join_kernel<T, 128>;
}

Kv8Plan kv8_prefill_plan(const vkq_kv8_cache &c, const vkq_kv8_batch &b, int dtype, int64_t heads, int causal,
                         int64_t window, int sms) {
    Kv8Plan q{};
    q.rows = dtype == VKQ_F32 ? 128 : 256;
    const int64_t g = heads / c.kv_heads;
    q.row_tiles = (int)((b.max_tokens * g + q.rows - 1) / q.rows);
    q.tiles = b.batch * c.kv_heads * q.row_tiles;
    int64_t keys = b.max_len;
    if (causal && window > 0) {
        const int64_t w = window + (q.rows + g - 1) / g + kKv8Block;
        if (w < keys) keys = w;
    }
    if (keys < 1) keys = 1;
    // Ranges: what is cheapest in units of a key tile's time (2.3 to 2.8 us), a
    // CTA an SM.  A CTA costs its key tiles (a causal tile sees all but half of
    // the new tokens on average) and kStart for its start and end; ranges cost
    // the join's launch and their parts' bytes.  Measured, 8 KV heads, bfloat16:
    // 512 rows of 65,536 keys (24 tiles) 1,377 us in one range, 362 in 4, 251 in
    // 6 (chosen), 347 in 8; 2,560 rows of 8,192 keys (80 tiles) 183, 151 in 3
    // (chosen), 236 in 16; 5,120 rows of 1,024 keys (160) 35 (chosen), 54 in 2.
    constexpr double kStart = 3., kJoin = 1.5, kPart = 0.019 / (256 * 128);
    const int64_t most = (keys + kPreKeys - 1) / kPreKeys;
    double seen = causal ? (double)keys - 0.5 * (double)(b.max_tokens < keys ? b.max_tokens : keys) : (double)keys;
    if (causal && window > 0) seen = (double)keys;
    int64_t best = most;  // a range's key tiles
    double least = 0.;
    for (int64_t n = 1; n <= 64 && n <= most; n++) {
        const int64_t tiles = (most + n - 1) / n, ranges = (most + tiles - 1) / tiles, ctas = q.tiles * ranges;
        double cost = (double)((ctas + sms - 1) / sms) * ((double)tiles * seen / (double)keys + kStart);
        if (ranges > 1) cost += kJoin + (double)(ctas * q.rows * c.head_dim) * kPart;
        if (n == 1 || cost < least) best = tiles, least = cost;
    }
    q.chunk = (int)(best * kPreKeys);
    q.splits = (int)((most + best - 1) / best);
    const bool moves = dtype != VKQ_F32 && q.chunk > (dtype == VKQ_F16 ? kMoveF16 : kMoveBf16);
    if (q.splits > 1 || moves) q.part_floats = (size_t)(q.tiles * q.splits * q.rows * c.head_dim);
    if (q.splits > 1) q.stat_floats = (size_t)(q.tiles * q.splits * q.rows * 2);
    return q;
}

cudaError_t kv8_prefill(const vkq_kv8_cache &c, int64_t layer, const vkq_kv8_batch &b, const Kv8AttentionArgs &a,
                        const Kv8Plan &q, cudaStream_t s) {
    PrefillParams p{};
    p.pool = kv8_pool(c, layer);
    p.batch = kv8_batch(b);
    p.q = a.q, p.out = a.out, p.qt = a.q_token, p.ot = a.out_token;
    p.heads = (int)a.heads, p.g = (int)(a.heads / c.kv_heads);
    p.row_tiles = q.row_tiles, p.splits = q.splits, p.chunk = q.chunk;
    p.f = a.scale * 1.4426950408889634f;
    p.causal = a.causal, p.window = a.causal ? (int)a.window : 0;
    const int size = act_bytes(a.dtype);
    p.vec = (((uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)(a.q_token * size) | (uintptr_t)(a.out_token * size)) & 15u) == 0;
    p.part = reinterpret_cast<float *>(static_cast<char *>(a.workspace) + kWorkspaceCounterHead);
    p.stat = p.part + q.part_floats;
    const void *fn = a.dtype == VKQ_F32   ? prefill_fn<float>(c.head_dim, p.pool.e4m3)
                     : a.dtype == VKQ_F16 ? prefill_fn<__half>(c.head_dim, p.pool.e4m3)
                                          : prefill_fn<__nv_bfloat16>(c.head_dim, p.pool.e4m3);
    const size_t smem = (size_t)((2 + kPreRing) * 2 + kPreRaw) * 128 * c.head_dim + 1024;
    cudaError_t e = kernel_smem(fn, smem, true);
    if (e != cudaSuccess) return e;
    // the warpgroups' register split draws on what the block is launched with
    static std::atomic<const void *> checked[12];
    std::atomic<const void *> &seen = checked[(a.dtype == VKQ_F32 ? 0 : a.dtype == VKQ_F16 ? 1 : 2) * 4 +
                                              (c.head_dim == 128 ? 2 : 0) + (p.pool.e4m3 ? 1 : 0)];
    if (seen.load() != fn) {
        cudaFuncAttributes fa;
        e = cudaFuncGetAttributes(&fa, fn);
        if (e != cudaSuccess) return e;
        if (fa.numRegs * kPreThreads < 512 * 128) return cudaErrorLaunchOutOfResources;
        seen.store(fn);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(q.tiles * q.splits));
    cfg.blockDim = dim3(kPreThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    void *args[] = {(void *)&p};
    e = cudaLaunchKernelExC(&cfg, fn, args);
    if (e != cudaSuccess || q.splits == 1) return e;
    cfg.gridDim = dim3((unsigned)(q.tiles * (q.rows / 32)));
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    const void *join = a.dtype == VKQ_F32   ? join_fn<float>(c.head_dim)
                       : a.dtype == VKQ_F16 ? join_fn<__half>(c.head_dim)
                                            : join_fn<__nv_bfloat16>(c.head_dim);
    return cudaLaunchKernelExC(&cfg, join, args);
}

int *kv8_prefill_status_word() { return status_word(g_kv8_prefill_status); }

}  // namespace vkq
