// Block quantizer and dequantizer of the 4-bit format.
//
// Both stream: a thread takes eight values at a time (16 bytes of the 16-bit side, 4 bytes of codes), and where the matrix is one long
// row, four times eight with all loads under way at once.  The quantizer's blocks of 32, 64 or 128 values are 4, 8 or 16 neighbouring
// lanes, which find the block's largest value by shuffles over the bits of |x|.
#include "int4_common.cuh"

#include <type_traits>

namespace bi8 {
namespace {

constexpr int kThreads = 256;

// Where the eight values of unit `i` lie: whole rows one behind the other need no division.
struct Unit {
    int64_t row;
    int64_t k;           // first value of the unit in its row
};
struct Rows {
    int64_t units, per_row;
    FastDiv div;         // by per_row, for fewer than 2^31 units
    bool small;
    int shift;           // a block is 1 << shift units
    Rows(int64_t M, int64_t K, int block)
        : units(M * ((K + block - 1) / block) * (block / 8)), per_row((K + block - 1) / block * (block / 8)), small(units < 0x7fffffffll),
          shift(block == 32 ? 2 : block == 64 ? 3 : 4) {
        if (small) div = FastDiv(per_row);
    }
    template <bool FLAT>
    __device__ __forceinline__ Unit unit(int64_t i) const {
        if (FLAT) return {0, i * 8};
        const int64_t row = small ? (int64_t)div.div((unsigned)i) : i / per_row;
        return {row, (i - row * per_row) * 8};
    }
};

// FLAT: K is a multiple of the block, rows and code rows are dense and aligned; the matrix is one long row.
template <bool FLAT>
constexpr int kUnits = FLAT ? 4 : 1;                 // of a thread

template <typename T, bool FLAT>
__global__ void __launch_bounds__(kThreads) quantize_int4_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q, int64_t ldq,
                                                                 T* __restrict__ s, int64_t K, Rows rows) {
    constexpr int N = kUnits<FLAT>;
    after_predecessor();
    const int64_t first = (int64_t)blockIdx.x * (N * kThreads) + threadIdx.x;
    uint4 v[N];
    Unit u[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int64_t i = first + n * kThreads;
        const bool live = i < rows.units;
        u[n] = live ? rows.unit<FLAT>(i) : Unit{0, 0};
        v[n] = make_uint4(0u, 0u, 0u, 0u);
        if (FLAT) {
            if (live) v[n] = ld_nc_v4(x + u[n].k);
        } else if (live) {
            const unsigned short* p = reinterpret_cast<const unsigned short*>(x) + u[n].row * ldx + u[n].k;
            uint32_t e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = u[n].k + j < K ? p[j] : 0u;
            v[n] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int64_t i = first + n * kThreads;
        uint32_t bits;
        const uint32_t w = quantize8<T>(v[n], 1 << rows.shift, &bits);
        if (i >= rows.units) continue;
        if (FLAT) {
            *reinterpret_cast<uint32_t*>(q + u[n].k / 2) = w;
        } else {
            uint8_t* p = q + u[n].row * ldq + u[n].k / 2;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (u[n].k + 2 * j < K) p[j] = (uint8_t)(w >> (8 * j));
        }
        if ((threadIdx.x & ((1 << rows.shift) - 1)) == 0) reinterpret_cast<unsigned short*>(s)[i >> rows.shift] = (unsigned short)bits;
    }
}

template <typename O>
__device__ __forceinline__ void store8(O* p, const float (&y)[8]);
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&y)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(y[0], y[1], y[2], y[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(y[4], y[5], y[6], y[7]);
}
template <>
__device__ __forceinline__ void store8<__half>(__half* p, const float (&y)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_f16x2(y[0], y[1]), pack_f16x2(y[2], y[3]), pack_f16x2(y[4], y[5]), pack_f16x2(y[6], y[7]));
}
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&y)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
}
template <typename O>
__device__ __forceinline__ O to_out(float y);
template <>
__device__ __forceinline__ float to_out<float>(float y) { return y; }
template <>
__device__ __forceinline__ __half to_out<__half>(float y) { return __float2half_rn(y); }
template <>
__device__ __forceinline__ __nv_bfloat16 to_out<__nv_bfloat16>(float y) { return __float2bfloat16_rn(y); }

template <typename T, typename O, bool FLAT>
__global__ void __launch_bounds__(kThreads) dequantize_int4_kernel(const uint8_t* __restrict__ q, int64_t ldq, const T* __restrict__ s,
                                                                   O* __restrict__ out, int64_t K, Rows rows) {
    constexpr int N = kUnits<FLAT>;
    after_predecessor();
    const int64_t first = (int64_t)blockIdx.x * (N * kThreads) + threadIdx.x;
    uint32_t w[N];
    float sc[N];
    Unit u[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int64_t i = first + n * kThreads;
        w[n] = kZeroCodes;
        sc[n] = 0.0f;
        if (i >= rows.units) continue;
        u[n] = rows.unit<FLAT>(i);
        sc[n] = F16Bits<T>::one(__ldg(reinterpret_cast<const unsigned short*>(s) + (i >> rows.shift)));
        if (FLAT) {
            w[n] = __ldg(reinterpret_cast<const uint32_t*>(q + u[n].k / 2));
        } else {
            const uint8_t* p = q + u[n].row * ldq + u[n].k / 2;
            w[n] = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (u[n].k + 2 * j < K) w[n] |= (uint32_t)p[j] << (8 * j);
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        if (first + n * kThreads >= rows.units) continue;
        float y[8];
        values8(sc[n], w[n], y);
        if (FLAT) {
            store8(out + u[n].k, y);
        } else {
            O* p = out + u[n].row * K + u[n].k;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (u[n].k + j < K) p[j] = to_out<O>(y[j]);
        }
    }
}

int grid_of(int64_t units, bool flat, unsigned* grid) {
    const int64_t per = (int64_t)kThreads * (flat ? kUnits<true> : kUnits<false>), g = (units + per - 1) / per;
    if (g > 0x7fffffff) return fail(BI8_ERR_LIMIT, "int4: %lld values exceed one launch", (long long)units * 8);
    *grid = (unsigned)g;
    return BI8_OK;
}

}  // namespace

int launch_quantize_int4(const void* x, int dt, int64_t ldx, uint8_t* q, int64_t ldq, void* s, int64_t M, int64_t K, int block, cudaStream_t st) {
    if (M == 0 || K == 0) return BI8_OK;
    const Rows rows(M, K, block);
    const bool flat = K % block == 0 && (M == 1 || (ldx == K && ldq == K / 2)) && aligned(x, 16) && aligned(q, 4);
    unsigned grid;
    if (int rc = grid_of(rows.units, flat, &grid)) return rc;
    auto go = [&](auto* tag, auto is_flat) {
        using T = std::remove_pointer_t<decltype(tag)>;
        return launch_chained(quantize_int4_kernel<T, decltype(is_flat)::value>, grid, kThreads, 0, st, static_cast<const T*>(x), ldx, q, ldq,
                              static_cast<T*>(s), K, rows);
    };
    auto by_layout = [&](auto* tag) { return flat ? go(tag, std::true_type{}) : go(tag, std::false_type{}); };
    return dt == BI8_BF16 ? by_layout(static_cast<__nv_bfloat16*>(nullptr)) : by_layout(static_cast<__half*>(nullptr));
}

int launch_dequantize_int4(const uint8_t* q, int64_t ldq, const void* s, int s_dt, void* out, int out_dt, int64_t M, int64_t K, int block,
                           cudaStream_t st) {
    if (M == 0 || K == 0) return BI8_OK;
    const Rows rows(M, K, block);
    const bool flat = K % block == 0 && (M == 1 || ldq == K / 2) && aligned(q, 4) && aligned(out, 16);
    unsigned grid;
    if (int rc = grid_of(rows.units, flat, &grid)) return rc;
    auto go = [&](auto* tag, auto* out_tag, auto is_flat) {
        using T = std::remove_pointer_t<decltype(tag)>;
        using O = std::remove_pointer_t<decltype(out_tag)>;
        return launch_chained(dequantize_int4_kernel<T, O, decltype(is_flat)::value>, grid, kThreads, 0, st, q, ldq, static_cast<const T*>(s),
                              static_cast<O*>(out), K, rows);
    };
    auto by_layout = [&](auto* tag, auto* o) { return flat ? go(tag, o, std::true_type{}) : go(tag, o, std::false_type{}); };
    auto by_out = [&](auto* tag) {
        if (out_dt == BI8_BF16) return by_layout(tag, static_cast<__nv_bfloat16*>(nullptr));
        if (out_dt == BI8_F16) return by_layout(tag, static_cast<__half*>(nullptr));
        return by_layout(tag, static_cast<float*>(nullptr));
    };
    return s_dt == BI8_BF16 ? by_out(static_cast<__nv_bfloat16*>(nullptr)) : by_out(static_cast<__half*>(nullptr));
}

}  // namespace bi8
