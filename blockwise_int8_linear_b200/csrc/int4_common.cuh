// What the kernels for 4-bit blocks share: the format, its arithmetic and the operand layouts of the tensor cores.
//
// Format: `block` consecutive values of a row have the scale s = max|x|, held exactly in x's own 16-bit type; a value's code is
// q = rint(7 x / s), -7 to 7, and stands for s q / 7.  A byte holds two neighbouring codes, offset by 8, the even one in its low half;
// a row of odd length ends in a code 0.  A block that holds an infinity or a NaN has the scale NaN: all of it reads as NaN.
#pragma once

#include "bi8_common.cuh"

#include <atomic>
#include <type_traits>

namespace bi8 {

constexpr int kCacheBlock = 64;          // values per block of a key/value cache

template <typename T>
struct F16Bits;
template <>
struct F16Bits<__nv_bfloat16> {
    static constexpr uint32_t kInf = 0x7f80u, kNaN = 0x7fc0u;
    __device__ static float lo(uint32_t w) { return bf16lo(w); }
    __device__ static float hi(uint32_t w) { return bf16hi(w); }
    __device__ static float one(uint32_t bits) { return __uint_as_float(bits << 16); }
    __device__ static uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
};
template <>
struct F16Bits<__half> {
    static constexpr uint32_t kInf = 0x7c00u, kNaN = 0x7e00u;
    __device__ static float lo(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w & 0xffffu))); }
    __device__ static float hi(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w >> 16))); }
    __device__ static float one(uint32_t bits) { return lo(bits); }
    __device__ static uint32_t pack(float a, float b) { return pack_f16x2(a, b); }
};

// Largest |value| among eight 16-bit values, as the bits of that type: without the sign they order like integers, NaN above infinity.
__device__ __forceinline__ uint32_t absmax8(const uint4& v) {
    const uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
    return max(m & 0xffffu, m >> 16);
}

// The codes of eight values under the scale `s` (finite): 32 bits, the first value's code in the lowest four.
//
// fma(x, 7/s, 56) lies between 49 and 63, where fp32 has steps of 2^-18: with 7/s good to 2^-23, a quotient 7x/s that is a tie k + 1/2 is
// off by at most 7 * 2^-23 before that rounding and lands on the tie, and any other is 2^-15 or more away from one (14x - (2k+1)s is a
// multiple of the smaller one's last place, for x >= s/14 and 11 significant bits), so it stays on its side.  Adding 1.5 * 2^23 then
// rounds to an integer, ties to even, whose bits are 0x4b400000 + 56 + q; eight of those times the powers of 16, less what is not q + 8,
// are the word.  Three operations a value, no division: 1/s is the hardware's estimate after one Newton step.  Very small and very
// large scales, whose reciprocal may leave the normal numbers, are moved to the middle first.
template <typename T>
__device__ __forceinline__ uint32_t codes8(const uint4& v, float s) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    auto word = [&](float r, auto value) {
        uint32_t out = 0u - 0x11111111u * (0x4b400000u + 56u - 8u);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            out += __float_as_uint(__fadd_rn(__fmaf_rn(value(i & 1 ? F16Bits<T>::hi(w[i / 2]) : F16Bits<T>::lo(w[i / 2])), r, 56.0f), 12582912.0f)) << (4 * i);
        return out;
    };
    if (s >= 0x1p-60f && s <= 0x1p100f) {
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
        r = __fmaf_rn(r, __fmaf_rn(-s, r, 1.0f), r);
        return word(7.0f * r, [](float x) { return x; });
    }
    const float lift = s < 1.0f ? 0x1p100f : 0x1p-100f;
    return word(s > 0.0f ? __fdiv_rn(7.0f, s * lift) : 0.0f, [lift](float x) { return x * lift; });
}
constexpr uint32_t kZeroCodes = 0x88888888u;

// Quantizes a block that lies in LANES neighbouring lanes, eight values each: codes of this lane, the scale's bits in all of them.  `lanes` are
// those that call together, whole blocks.
template <typename T, int LANES>
__device__ __forceinline__ uint32_t quantize8(const uint4& v, uint32_t lanes, uint32_t* scale_bits) {
    uint32_t m = absmax8(v);
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) m = max(m, __shfl_xor_sync(lanes, m, d));
    const bool bad = m >= F16Bits<T>::kInf;
    *scale_bits = bad ? F16Bits<T>::kNaN : m;
    return bad ? kZeroCodes : codes8<T>(v, F16Bits<T>::one(m));
}

// s q / 7 in fp32, rounded once, for the codes q of a word under one scale.  With 1/7 = h + l and s h = a + e exactly (a rounded, e its error),
// s q / 7 = q a + q (e + s l): the first product is exact inside a multiply-add, the second is 2^-24 of it and its rounding harmless.
// Scales outside the range in which e is exact take the division itself, the largest a factor of 2^20 lower, where 7 s does not overflow.
__device__ __forceinline__ void values8(float s, uint32_t w, float (&y)[8]);

// ---- tensor-core operands -----------------------------------------------------------------------------------------------------
// Codes become the matrix instruction's operands in pairs, as numbers in the other operand's type: -7 to 7 in fp16, and 2^-10 of that in bf16
// (kCodeUnit), where a block's sum of codes times values as large as the type has would overflow otherwise.  Four bits c + 8 under the
// exponent of 1024 are the fp16 number 1024 + 8 + c, four bits further up 1024 + 16 (8 + c); a packed subtraction or multiply-add
// makes c of them, exactly: eight codes are one shift, four AND-ORs and four packed operations.  bf16 has (128 + 8 + c) 2^-10, and no room for
// four bits further up: two shifts more.  (This way of unpacking is the usual one of kernels with 4-bit weights.  The four bits alone are fp16 denormals, (8 + c) 2^-24, and the offset could be left to the
// accumulator's start value, which saves half of that.  But the instruction aligns its sums by the operands' exponent fields, and ten
// leading zeros in one operand cost the sum as many bits: measured, 2^-16 of the largest term.)
//
// Order of a word's eight codes in the contraction: pairs (0,4), (1,5), (2,6), (3,7).
struct Codes4 {
    uint32_t p04, p15, p26, p37;
};
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t set) {      // (w & mask) | set, as one instruction: the compiler makes two of it
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(set));
    return r;
}
__device__ __forceinline__ uint32_t half2_low(uint32_t w) {
    const uint32_t v = and_or(w, 0x000f000fu, 0x64006400u), k = 0x64086408u;              // 1024 + 8 + c, 1032
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&k));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t half2_high(uint32_t w) {
    const uint32_t v = and_or(w, 0x00f000f0u, 0x64006400u), m = 0x2c002c00u, k = 0xd480d480u;      // 1024 + 16 (8 + c), 1/16, -72
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&m), *reinterpret_cast<const __half2*>(&k));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t bf162_low(uint32_t w) {
    const uint32_t v = and_or(w, 0x000f000fu, 0x3e003e00u), k = 0x3e083e08u;              // (128 + 8 + c) 2^-10, 136 * 2^-10
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&k));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <typename T>
constexpr float kCodeUnit = std::is_same<T, __half>::value ? 1.0f : 0x1p-10f;           // what a code of 1 becomes
template <typename T>
__device__ __forceinline__ Codes4 unpack8(uint32_t w) {
    if (std::is_same<T, __half>::value) return {half2_low(w), half2_high(w), half2_low(w >> 8), half2_high(w >> 8)};
    return {bf162_low(w), bf162_low(w >> 4), bf162_low(w >> 8), bf162_low(w >> 12)};
}
__device__ __forceinline__ void values8(float s, uint32_t w, float (&y)[8]) {
    constexpr float H = 1.0f / 7.0f, L = (float)(1.0 / 7.0 - (double)H);
    const Codes4 c = unpack8<__half>(w);
    const uint32_t pairs[4] = {c.p04, c.p15, c.p26, c.p37};
    if ((s > 0x1p-90f && s < 0x1p127f) || s == 0.0f) {
        const float a = s * H, b = __fmaf_rn(s, L, __fmaf_rn(s, H, -a));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float q = i < 4 ? F16Bits<__half>::lo(pairs[i]) : F16Bits<__half>::hi(pairs[i - 4]);
            y[i] = __fmaf_rn(q, a, q * b);
        }
    } else {
        const float up = s > 1.0f ? 0x1p20f : 1.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __fdiv_rn(s / up * (i < 4 ? F16Bits<__half>::lo(pairs[i]) : F16Bits<__half>::hi(pairs[i - 4])), 7.0f) * up;
    }
}
// Eight neighbouring 16-bit values in that order.
__device__ __forceinline__ uint4 paired8(const uint4& v) {
    return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
}

// D = C + A B, A 16 x 16 (rows g and g + 8 of lane 4 g + c, columns 2c, 2c+1 and 2c+8, 2c+9), B 16 x 8 (column g), C and D 16 x 8 (columns
// 2c, 2c+1)
template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1,
                                      float c2, float c3) {
    if (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {      // D += A B
    mma16<T>(d, a0, a1, a2, a3, b0, b1, d[0], d[1], d[2], d[3]);
}
template <typename T>
__device__ __forceinline__ void mma16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {      // D = A B
    mma16<T>(d, a0, a1, a2, a3, b0, b1, 0.0f, 0.0f, 0.0f, 0.0f);
}

// ---- asynchronous copies into shared memory ----------------------------------------------------------------------------------
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {      // bytes read; the rest of the 16 is zero
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void copy_some(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void wait_copies() {
    asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// SMs of the current device.
inline int sm_count() {
    static std::atomic<int> sms[64];             // calls come from several threads
    int dev = 0;
    if (current_device(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    int n = sms[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) n = 148;
        sms[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

}  // namespace bi8
