// rotary.cuh -- one thread's item of a rotation, shared by vkq_rotary and the
// cache's append (which rotates q beside the keys).
#pragma once

#include "act.cuh"

namespace vkq {

constexpr int kRotHeads = 4;  // heads of a token that share an item's table entries

// The vector path: heads in 16-byte pieces of V elements, rot a multiple of
// 2V, aligned rows.  Interleaved: piece j of D / V (the rotated ones first);
// half: the rot / 2V partner pairs, then the pieces past rot by twos (every
// item moves two).
template <typename T>
__host__ __device__ __forceinline__ int rotary_pieces(int D, int rot, bool half) {
    const int V = 16 / (int)sizeof(T);
    return half ? rot / (2 * V) + ((D - rot) / V + 1) / 2 : D / V;
}
// Whether rows at these addresses and strides (in bytes, or'ed) and this rot take it.
inline bool rotary_vec(uintptr_t bits, int64_t rot) { return (bits & 15u) == 0 && rot % 16 == 0; }

// Piece j of up to kRotHeads heads from x to o (head strides xh, oh); `row()`
// gives the position, or a negative number to leave the item out.  The heads
// are under way before it is asked.  o may be x.
template <typename T, bool HALF, typename Row>
__device__ __forceinline__ void rotary_item(const T *x, int64_t xh, T *o, int64_t oh, int heads, int j, int D, int rot,
                                            const float *cos_t, const float *sin_t, bool inverse, Row row) {
    constexpr int V = 16 / (int)sizeof(T);
    constexpr int NP = HALF ? V : V / 2;  // pairs of an item
    const int turned = HALF ? rot / (2 * V) : rot / V;
    const bool turns = j < turned;
    // first element of the piece, and of its partner
    const int a0 = HALF && !turns ? rot + (j - turned) * 2 * V : j * V;
    const int b0 = !HALF ? a0 : turns ? a0 + rot / 2 : a0 + V;
    const bool two = HALF && b0 < D;  // all but a last odd piece
    uint4 a[kRotHeads], b[kRotHeads];
#pragma unroll
    for (int u = 0; u < kRotHeads; u++) {
        if (u < heads) {
            a[u] = *reinterpret_cast<const uint4 *>(x + u * xh + a0);
            if (two) b[u] = *reinterpret_cast<const uint4 *>(x + u * xh + b0);
        }
    }
    const int64_t ps = row();
    if (ps < 0) return;
    if (!turns) {
#pragma unroll
        for (int u = 0; u < kRotHeads; u++) {
            if (u >= heads) break;
            *reinterpret_cast<uint4 *>(o + u * oh + a0) = a[u];
            if (two) *reinterpret_cast<uint4 *>(o + u * oh + b0) = b[u];
        }
        return;
    }
    float c[NP], s[NP];
    const int64_t e = ps * (rot / 2) + (HALF ? a0 : a0 / 2);
    load_act<float, NP>(cos_t + e, c, true);
    load_act<float, NP>(sin_t + e, s, true);
    if (inverse)
#pragma unroll
        for (int i = 0; i < NP; i++) s[i] = -s[i];
#pragma unroll
    for (int u = 0; u < kRotHeads; u++) {
        if (u >= heads) break;
        const T *xa = reinterpret_cast<const T *>(&a[u]), *xb = reinterpret_cast<const T *>(&b[u]);
        float fa[V], fb[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            fa[i] = to_f32<T>(xa[i]);
            if constexpr (HALF) fb[i] = to_f32<T>(xb[i]);
        }
#pragma unroll
        for (int i = 0; i < NP; i++) {
            if constexpr (HALF) turn(fa[i], fb[i], c[i], s[i]);
            else turn(fa[2 * i], fa[2 * i + 1], c[i], s[i]);
        }
        store_act<T, V>(o + u * oh + a0, fa, true);
        if constexpr (HALF) store_act<T, V>(o + u * oh + b0, fb, true);
    }
}

// Any rot, strides and alignment: item j of a head's D - rot / 2 is one pair, or
// one value past rot.
template <typename T>
__device__ __forceinline__ void rotary_one(const T *x, T *o, int j, int rot, bool half, const float *cos_t,
                                           const float *sin_t, bool inverse, int64_t ps) {
    const int h = rot / 2;
    if (j >= h) {
        o[h + j] = x[h + j];
        return;
    }
    const int ia = half ? j : 2 * j, ib = half ? j + h : 2 * j + 1;
    const int64_t e = ps * h + j;
    float a = to_f32<T>(x[ia]), b = to_f32<T>(x[ib]);
    const float s = sin_t[e];
    turn(a, b, cos_t[e], inverse ? -s : s);
    o[ia] = from_f32<T>(a);
    o[ib] = from_f32<T>(b);
}

}  // namespace vkq
