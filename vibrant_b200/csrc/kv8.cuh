// kv8.cuh -- the 8-bit paged KV cache as its kernels see it: the batch's
// sequences, where a block of 16 tokens lies, codes to values and back.
//
// A value is code * scale with one scale for the 16 tokens of a block and one
// KV head.  Codes are int8 or e4m3; both are exact in float16 (8 and 4
// significant bits, magnitudes up to 127 and 448), so a matrix instruction
// with float16 operands multiplies them without rounding and the scales go
// into the scores (K) and the probabilities' sums (V) in float32.
#pragma once

#include <cstdint>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "../../include/vkq.h"
#include "kq_device.cuh"

namespace vkq {

constexpr int kKv8Block = VKQ_KV8_BLOCK;
constexpr float kKv8MinScale = 5.421010862427522e-20f;  // 2^-64
constexpr float kKv8MaxScale = 9.223372036854775808e18f;  // 2^63

// One layer of the pool.
struct Kv8Pool {
    uint8_t *k, *v;      // [num_pages][kv_heads][page][D]
    float *ks, *vs;      // [num_pages][kv_heads][page / 16]
    int64_t num_pages;
    int kv_heads, page, D;
    bool e4m3;
};

inline Kv8Pool kv8_pool(const vkq_kv8_cache &c, int64_t layer) {
    const int64_t codes = c.num_pages * c.kv_heads * c.page_size * c.head_dim;
    const int64_t scales = c.num_pages * c.kv_heads * (c.page_size / kKv8Block);
    return Kv8Pool{static_cast<uint8_t *>(c.k) + layer * codes, static_cast<uint8_t *>(c.v) + layer * codes,
                   c.k_scale + layer * scales, c.v_scale + layer * scales, c.num_pages,
                   c.kv_heads, c.page_size, c.head_dim, c.format == VKQ_KV8_E4M3};
}

struct Kv8Batch {
    const int *table, *lens, *slots, *cu;
    int64_t rows, max_pages, batch, tokens, max_tokens, max_len;
};

inline Kv8Batch kv8_batch(const vkq_kv8_batch &b) {
    return Kv8Batch{b.table, b.lens, b.slots, b.cu_tokens, b.rows, b.max_pages, b.batch, b.tokens, b.max_tokens, b.max_len};
}

// A sequence of the batch: its table row, its length, the row of its first new
// token in q/k/v/out and how many there are.  ok: everything in bounds.
struct Kv8Seq {
    const int *pages;
    int len, first, n;
    bool ok;
};

__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8Batch &b, int page, int64_t i) {
    Kv8Seq s{};
    // all loads first (the row clamped for the length's), then the checks
    const int64_t c0 = b.cu ? b.cu[i] : i, c1 = b.cu ? b.cu[i + 1] : i + 1;
    const int64_t r = b.slots ? b.slots[i] : i;
    const int64_t in = r < 0 ? 0 : r < b.rows ? r : b.rows - 1;
    const int len = b.lens[in];
    s.ok = c0 >= 0 && c1 >= c0 && c1 <= b.tokens && c1 - c0 <= b.max_tokens;
    if (!s.ok) return s;  // n == 0: no rows of this sequence are known
    s.first = (int)c0;
    s.n = (int)(c1 - c0);
    s.ok = r == in && len >= 0 && len <= b.max_len && len <= b.max_pages * page;
    s.pages = b.table + in * b.max_pages;
    s.len = len;
    return s;
}

// The page of logical page lp (within the sequence's length), -1 if the table holds none.
__device__ __forceinline__ int kv8_page(const Kv8Pool &p, const Kv8Seq &s, int lp) {
    const int id = s.pages[lp];
    return id >= 0 && id < p.num_pages ? id : -1;
}

// x / d for d >= 1 by a multiplication: `magic` is floor((2^32 - 1) / d) + 1 (0
// for d = 1), the quotient then at most one too large.
inline uint32_t kv8_magic(uint32_t d) { return d == 1 ? 0u : 0xffffffffu / d + 1u; }
__device__ __forceinline__ uint32_t kv8_div(uint32_t x, uint32_t d, uint32_t magic) {
    uint32_t q = magic ? __umulhi(x, magic) : x;
    if (q * d > x) q--;
    return q;
}

// ---- codes ----------------------------------------------------------------
__device__ __forceinline__ float kv8_decode(uint32_t byte, bool e4m3) {
    if (e4m3) {
        const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3);
        return __half2float(__half(h));
    }
    return (float)(int8_t)byte;
}
// Nearest code, ties to even, saturating; NaN gives 0.
__device__ __forceinline__ uint32_t kv8_encode(float x, bool e4m3) {
    if (!(x == x)) x = 0.f;
    if (e4m3) return __nv_cvt_float_to_fp8(fminf(fmaxf(x, -448.f), 448.f), __NV_SATFINITE, __NV_E4M3);
    return (uint32_t)(uint8_t)(int8_t)__float2int_rn(fminf(fmaxf(x, -127.f), 127.f));
}
// Four codes of values within the format's range (finite, |x| <= 448 or 127).
__device__ __forceinline__ uint32_t kv8_encode4(float a, float b, float c, float d, bool e4m3) {
    if (e4m3) {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
        return (uint32_t)lo | ((uint32_t)hi << 16);
    }
    // adding 1.5 * 2^23 leaves the integer (ties to even) in the low bits
    const float m = 12582912.f;
    const uint32_t x = __float_as_uint(__fadd_rn(a, m)), y = __float_as_uint(__fadd_rn(b, m));
    const uint32_t z = __float_as_uint(__fadd_rn(c, m)), w = __float_as_uint(__fadd_rn(d, m));
    return prmt(prmt(x, y, 0x0040u), prmt(z, w, 0x0040u), 0x5410u);
}
// The least power of two s in [2^-64, 2^63] with a <= m * s (a finite, >= 0).
__device__ __forceinline__ float kv8_scale(float a, bool e4m3) {
    const float m = e4m3 ? 448.f : 127.f;
    const int top = e4m3 ? 8 : 6;  // 2^top <= m < 2^(top + 1)
    a = fmaxf(a, 1e-30f);
    const int e = (int)(__float_as_uint(a) >> 23) - 127 - top;  // a normal: 2^(e + top) <= a
    float s = __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
    if (a > m * s) s *= 2.f;
    return fminf(fmaxf(s, kKv8MinScale), kKv8MaxScale);
}

// Codes as float16 pairs, exactly.  int8: the byte with its sign bit flipped
// (kv8_unsign) is the low byte of 1024 + 128 + code.  e4m3: the hardware's
// conversion (0x7f and 0xff, which are no codes, give NaN).
template <bool E4M3> __device__ __forceinline__ uint32_t kv8_unsign(uint32_t w) { return E4M3 ? w : w ^ 0x80808080u; }
// Bytes (0, 1) or (2, 3) of an unsigned word.
template <bool E4M3, bool HIGH>
__device__ __forceinline__ uint32_t kv8_widen(uint32_t w) {
    if constexpr (E4M3) {
        uint32_t r;
        if constexpr (HIGH) asm("{ .reg .b16 a, b; mov.b32 {a, b}, %1; cvt.rn.f16x2.e4m3x2 %0, b; }" : "=r"(r) : "r"(w));
        else asm("{ .reg .b16 a, b; mov.b32 {a, b}, %1; cvt.rn.f16x2.e4m3x2 %0, a; }" : "=r"(r) : "r"(w));
        return r;
    } else {
        const uint32_t u = prmt(w, 0x64646464u, HIGH ? 0x4342u : 0x4140u);
        const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&u), __half2half2(__ushort_as_half(0x6480)));
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

}  // namespace vkq
