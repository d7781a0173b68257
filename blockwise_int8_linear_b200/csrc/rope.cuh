// Rotary positions: the arithmetic that the standalone operator and the paged cache's append share.
//
// A pair of features (x, y) is turned by the angle of its position: (x c - y s, x s + y c), fp32 products and sums each rounded on their own, the
// result rounded to the activations' type.  Pairs are neighbours (interleaved) or lie half of the rotated features apart (half).
//
// A thread takes two pieces of P features of a head, the first from the lower half of the rotated features and the other as far into the
// upper one.  So the addresses are the same in both layouts: in one of them the pieces are the two sides of P pairs, in the other each
// has P / 2 pairs of its own.  Neighbouring threads read neighbouring pieces.  Features that are not rotated come in two pieces as well.
#pragma once

#include "int4_common.cuh"

namespace bi8 {

template <typename T>
struct RopeType {                        // the two 16-bit types: two values to a word
    static constexpr int kPerWord = 2;
    static __device__ __forceinline__ float get(uint32_t w, int i) { return i ? F16Bits<T>::hi(w) : F16Bits<T>::lo(w); }
    static __device__ __forceinline__ uint32_t set(float a, float b) { return F16Bits<T>::pack(a, b); }
};
template <>
struct RopeType<float> {
    static constexpr int kPerWord = 1;
    static __device__ __forceinline__ float get(uint32_t w, int) { return __uint_as_float(w); }
    static __device__ __forceinline__ uint32_t set(float a, float) { return __float_as_uint(a); }
};

// P values as they lie in memory, read and written 16 bytes at a time where they have as many.
template <typename T, int P>
struct Piece {
    static constexpr int kWords = P / RopeType<T>::kPerWord;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kWords == 1) {
            w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
        } else if constexpr (kWords == 2) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
            w[0] = v.x, w[1] = v.y;
        } else {
#pragma unroll
            for (int i = 0; i < kWords; i += 4) {
                const uint4 v = ld_nc_v4(p + i * RopeType<T>::kPerWord);
                w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
            }
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (kWords == 1) {
            *reinterpret_cast<uint32_t*>(p) = w[0];
        } else if constexpr (kWords == 2) {
            *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int i = 0; i < kWords; i += 4) *reinterpret_cast<uint4*>(p + i * RopeType<T>::kPerWord) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0u;
    }
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
    using R = RopeType<T>;
    constexpr int N = R::kPerWord;
    if (half_layout) {
#pragma unroll
        for (int k = 0; k < P / N; ++k) {
            float x[2] = {}, y[2] = {};
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x[i] = R::get(a.w[k], i), y[i] = R::get(b.w[k], i);
                turn(x[i], y[i], g.c[N * k + i], g.s[N * k + i]);
            }
            a.w[k] = R::set(x[0], x[1]);
            b.w[k] = R::set(y[0], y[1]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < P / 2; ++k) {                     // a pair of either piece
            constexpr int STEP = 2 / N;
#pragma unroll
            for (int side = 0; side < 2; ++side) {
                Piece<T, P>& p = side ? b : a;
                float x = R::get(p.w[k * STEP], 0), y = R::get(p.w[k * STEP + STEP - 1], 1);
                turn(x, y, g.c[side * (P / 2) + k], g.s[side * (P / 2) + k]);
                p.w[k * STEP] = R::set(x, y);
                if (N == 1) p.w[k * STEP + STEP - 1] = R::set(y, y);
            }
        }
    }
}

}  // namespace bi8
