// Rotary positions: the arithmetic that the standalone operator and the paged cache's append share.
//
// A pair of features (x, y) is turned by the angle of its position: (x c - y s, x s + y c), fp32 products and sums each rounded on their own, the
// result rounded to the activations' type.  Pairs are neighbours (interleaved) or lie half of the rotated features apart (half).
//
// A thread takes two pieces of P features of a head, the first from the lower half of the rotated features and the other as far into the
// upper one.  So the addresses are the same in both layouts: in one of them the pieces are the two sides of P pairs, in the other each
// has P / 2 pairs of its own.  Neighbouring threads read neighbouring pieces.  Features that are not rotated come in two pieces as well.
#pragma once

#include "bi8_common.cuh"

namespace bi8 {

// P values of a type as floats, and back with one rounding.  P * sizeof(T) bytes are read at a time, up to 16.
template <typename T>
struct RopeType;
template <>
struct RopeType<float> {
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float set(float v) { return v; }
};
template <>
struct RopeType<__nv_bfloat16> {
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 set(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct RopeType<__half> {
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half set(float v) { return __float2half_rn(v); }
};

template <typename T, int P>
struct alignas(sizeof(T) * P > 16 ? 16 : sizeof(T) * P) Piece {
    T v[P];
};

template <int P>
struct Angles {
    float c[P], s[P];
};

// Where the pieces of unit u (of D / 2P) begin.  R and D are multiples of 2P.
template <int P>
__device__ __forceinline__ void piece_offsets(int u, int R, int D, int& a, int& b) {
    const int turned = R / (2 * P);
    a = u < turned ? u * P : R + (u - turned) * P;
    b = a + (u < turned ? R / 2 : (D - R) / 2);
}

// The angles of unit u < R / 2P at one table row: R / 2 pairs, on a 16-byte boundary where P is 4 or more.
template <int P>
__device__ __forceinline__ Angles<P> load_angles(const float2* row, int u, int R, bool half_layout) {
    Angles<P> g;
    const float2* const first = row + (half_layout ? u * P : u * (P / 2));
    const float2* const second = half_layout ? first + P / 2 : first + R / 4;
    if constexpr (P >= 4) {
#pragma unroll
        for (int j = 0; j < P / 2; j += 2) {
            const float4 x = __ldg(reinterpret_cast<const float4*>(first + j)), y = __ldg(reinterpret_cast<const float4*>(second + j));
            g.c[j] = x.x, g.s[j] = x.y, g.c[j + 1] = x.z, g.s[j + 1] = x.w;
            g.c[P / 2 + j] = y.x, g.s[P / 2 + j] = y.y, g.c[P / 2 + j + 1] = y.z, g.s[P / 2 + j + 1] = y.w;
        }
    } else {
        const float2 x = __ldg(first), y = __ldg(second);
        g.c[0] = x.x, g.s[0] = x.y, g.c[1] = y.x, g.s[1] = y.y;
    }
    return g;
}

__device__ __forceinline__ void turn(float& x, float& y, float c, float s) {
    const float a = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s)), b = __fadd_rn(__fmul_rn(x, s), __fmul_rn(y, c));
    x = a;
    y = b;
}

template <typename T, int P>
__device__ __forceinline__ void turn_pieces(Piece<T, P>& a, Piece<T, P>& b, const Angles<P>& g, bool half_layout) {
    float x[P], y[P];
#pragma unroll
    for (int j = 0; j < P; ++j) {
        x[j] = RopeType<T>::get(a.v[j]);
        y[j] = RopeType<T>::get(b.v[j]);
    }
    if (half_layout) {
#pragma unroll
        for (int j = 0; j < P; ++j) turn(x[j], y[j], g.c[j], g.s[j]);
    } else {
#pragma unroll
        for (int j = 0; j < P / 2; ++j) {
            turn(x[2 * j], x[2 * j + 1], g.c[j], g.s[j]);
            turn(y[2 * j], y[2 * j + 1], g.c[P / 2 + j], g.s[P / 2 + j]);
        }
    }
#pragma unroll
    for (int j = 0; j < P; ++j) {
        a.v[j] = RopeType<T>::set(x[j]);
        b.v[j] = RopeType<T>::set(y[j]);
    }
}

}  // namespace bi8
