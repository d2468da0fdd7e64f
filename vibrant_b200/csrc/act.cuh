// act.cuh -- activations of the serving kernels: float32, float16 or bfloat16
// elements in memory, float32 in registers.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/vkq.h"

namespace vkq {

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N consecutive elements, as N * sizeof(T) / 16 vectors of 16 bytes (or one of
// 8 or 4) when `vec` (the address is aligned for it), else one by one.
template <typename T, int N>
__device__ __forceinline__ void load_act(const T *p, float (&r)[N], bool vec) {
    constexpr int BYTES = N * (int)sizeof(T);
    if (vec) {
        alignas(16) T t[N];
        if constexpr (BYTES % 16 == 0) {
#pragma unroll
            for (int i = 0; i < BYTES / 16; i++)
                reinterpret_cast<uint4 *>(t)[i] = reinterpret_cast<const uint4 *>(p)[i];
        } else if constexpr (BYTES == 8) {
            *reinterpret_cast<uint2 *>(t) = *reinterpret_cast<const uint2 *>(p);
        } else {
            static_assert(BYTES == 4, "4, 8 or a multiple of 16 bytes");
            *reinterpret_cast<uint32_t *>(t) = *reinterpret_cast<const uint32_t *>(p);
        }
#pragma unroll
        for (int i = 0; i < N; i++) r[i] = to_f32<T>(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) r[i] = to_f32<T>(p[i]);
    }
}

template <typename T, int N>
__device__ __forceinline__ void store_act(T *p, const float (&r)[N], bool vec) {
    constexpr int BYTES = N * (int)sizeof(T);
    if (vec) {
        alignas(16) T t[N];
#pragma unroll
        for (int i = 0; i < N; i++) t[i] = from_f32<T>(r[i]);
        if constexpr (BYTES % 16 == 0) {
#pragma unroll
            for (int i = 0; i < BYTES / 16; i++)
                reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(t)[i];
        } else if constexpr (BYTES == 8) {
            *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(t);
        } else {
            static_assert(BYTES == 4, "4, 8 or a multiple of 16 bytes");
            *reinterpret_cast<uint32_t *>(p) = *reinterpret_cast<const uint32_t *>(t);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) p[i] = from_f32<T>(r[i]);
    }
}

// A pair turned by (c, s): each product and sum rounded on its own (the
// arithmetic of vkq_rope_f32).
__device__ __forceinline__ void turn(float &a, float &b, float c, float s) {
    const float x = a, y = b;
    a = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
    b = __fadd_rn(__fmul_rn(x, s), __fmul_rn(y, c));
}

inline int act_bytes(int dtype) { return dtype == VKQ_F32 ? 4 : dtype == VKQ_F16 || dtype == VKQ_BF16 ? 2 : 0; }

}  // namespace vkq
