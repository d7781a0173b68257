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

// Eight 16-bit values from any address, those from `count` (below 1: all) on as zeros: from the two aligned 16 bytes that hold them, each read
// only where it holds one of them.
__device__ __forceinline__ uint4 load8(const unsigned short* p, int count) {
    if (count < 1) return make_uint4(0u, 0u, 0u, 0u);
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), base = a & ~(uintptr_t)15;
    const uint4 lo = __ldg(reinterpret_cast<const uint4*>(base));
    uint4 hi = make_uint4(0u, 0u, 0u, 0u);
    if (base + 16 < a + 2 * count) hi = __ldg(reinterpret_cast<const uint4*>(base + 16));
    const uint32_t r[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    const uint32_t words = (uint32_t)(a & 15u) >> 2, bits = (uint32_t)(a & 2u) * 8u;
    uint32_t w[5];
#pragma unroll
    for (int j = 0; j < 5; ++j) w[j] = words & 2u ? (j + 2 < 8 ? r[j + 2] : 0u) : r[j];
    const uint32_t next = words & 2u ? r[7] : r[5];
    uint32_t v[5];
#pragma unroll
    for (int j = 0; j < 5; ++j) v[j] = words & 1u ? (j + 1 < 5 ? w[j + 1] : next) : w[j];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[j] = __funnelshift_r(v[j], v[j + 1], bits);
        v[j] = 2 * j + 1 < count ? v[j] : 2 * j < count ? v[j] & 0xffffu : 0u;
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

template <typename T, bool FLAT, int LANES>
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
            v[n] = load8(reinterpret_cast<const unsigned short*>(x) + u[n].row * ldx + u[n].k, (int)min((int64_t)8, K - u[n].k));
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int64_t i = first + n * kThreads;
        uint32_t bits;
        const uint32_t w = quantize8<T, LANES>(v[n], 0xffffffffu, &bits);
        if (i >= rows.units) continue;
        if (FLAT) {
            *reinterpret_cast<uint32_t*>(q + u[n].k / 2) = w;
        } else {
            uint8_t* p = q + u[n].row * ldq + u[n].k / 2;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (u[n].k + 2 * j < K) p[j] = (uint8_t)(w >> (8 * j));
        }
        if (threadIdx.x % LANES == 0) reinterpret_cast<unsigned short*>(s)[i / LANES] = (unsigned short)bits;
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

template <typename T, typename O>
__global__ void __launch_bounds__(kThreads) dequantize_int4_kernel(const uint8_t* __restrict__ q, const T* __restrict__ s, O* __restrict__ out, Rows rows) {
    constexpr int N = kUnits<true>;
    after_predecessor();
    const int64_t first = (int64_t)blockIdx.x * (N * kThreads) + threadIdx.x;
    uint32_t w[N];
    float sc[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int64_t i = first + n * kThreads;
        w[n] = kZeroCodes;
        sc[n] = 0.0f;
        if (i >= rows.units) continue;
        sc[n] = F16Bits<T>::one(__ldg(reinterpret_cast<const unsigned short*>(s) + (i >> rows.shift)));
        w[n] = __ldg(reinterpret_cast<const uint32_t*>(q) + i);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int64_t i = first + n * kThreads;
        if (i >= rows.units) continue;
        float y[8];
        values8(sc[n], w[n], y);
        store8(out + i * 8, y);
    }
}

// Rows of any length and alignment: a warp takes 256 neighbouring values of a row, a lane every 32nd, so that what the lanes store at a time
// lies together.
template <typename T, typename O>
__global__ void __launch_bounds__(kThreads) dequantize_int4_rows_kernel(const uint8_t* __restrict__ q, int64_t ldq, const T* __restrict__ s, O* __restrict__ out,
                                                                        int64_t K, int64_t blocks, Rows rows) {
    after_predecessor();
    const int64_t warp = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    if (warp >= rows.units) return;
    const Unit u = rows.unit<false>(warp);                      // a unit of 256 values
    const int64_t k0 = u.k * 32 + (threadIdx.x & 31), left = K - k0;
    const uint8_t* const codes = q + u.row * ldq + k0 / 2;
    const unsigned short* const scales = reinterpret_cast<const unsigned short*>(s) + u.row * blocks + (k0 >> rows.shift);
    O* const to = out + u.row * K + k0;
    const uint32_t nibble = k0 & 1 ? 4u : 0u;
    uint32_t byte[8], bits[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (32 * j < left) byte[j] = __ldg(codes + 16 * j), bits[j] = __ldg(scales + ((32 * j) >> rows.shift));      // k0 - lane is a multiple of 256
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (32 * j < left) {
            float y[8];
            values8(F16Bits<T>::one(bits[j]), byte[j] >> nibble, y);        // the first one counts
            to[32 * j] = to_out<O>(y[0]);
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
    auto go = [&](auto* tag, auto is_flat, auto lanes) {
        using T = std::remove_pointer_t<decltype(tag)>;
        return launch_chained(quantize_int4_kernel<T, decltype(is_flat)::value, decltype(lanes)::value>, grid, kThreads, 0, st, static_cast<const T*>(x), ldx, q, ldq,
                              static_cast<T*>(s), K, rows);
    };
    auto by_block = [&](auto* tag, auto is_flat) {
        if (block == 32) return go(tag, is_flat, std::integral_constant<int, 4>{});
        if (block == 64) return go(tag, is_flat, std::integral_constant<int, 8>{});
        return go(tag, is_flat, std::integral_constant<int, 16>{});
    };
    auto by_layout = [&](auto* tag) { return flat ? by_block(tag, std::true_type{}) : by_block(tag, std::false_type{}); };
    return dt == BI8_BF16 ? by_layout(static_cast<__nv_bfloat16*>(nullptr)) : by_layout(static_cast<__half*>(nullptr));
}

int launch_dequantize_int4(const uint8_t* q, int64_t ldq, const void* s, int s_dt, void* out, int out_dt, int64_t M, int64_t K, int block,
                           cudaStream_t st) {
    if (M == 0 || K == 0) return BI8_OK;
    const Rows rows(M, K, block);
    const bool flat = K % block == 0 && (M == 1 || ldq == K / 2) && aligned(q, 4) && aligned(out, 16);
    Rows pieces = rows;                                     // of 256 values, for a warp each
    pieces.per_row = (K + 255) / 256;
    pieces.units = M * pieces.per_row;
    pieces.small = pieces.units < 0x7fffffffll;
    pieces.shift = rows.shift + 3;                          // a block in values
    if (pieces.small) pieces.div = FastDiv(pieces.per_row);
    unsigned grid;
    if (int rc = grid_of(flat ? rows.units : pieces.units * 32, flat, &grid)) return rc;
    auto by_layout = [&](auto* tag, auto* out_tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        using O = std::remove_pointer_t<decltype(out_tag)>;
        if (flat) return launch_chained(dequantize_int4_kernel<T, O>, grid, kThreads, 0, st, q, static_cast<const T*>(s), static_cast<O*>(out), rows);
        return launch_chained(dequantize_int4_rows_kernel<T, O>, grid, kThreads, 0, st, q, ldq, static_cast<const T*>(s), static_cast<O*>(out), K,
                              (K + block - 1) / block, pieces);
    };
    auto by_out = [&](auto* tag) {
        if (out_dt == BI8_BF16) return by_layout(tag, static_cast<__nv_bfloat16*>(nullptr));
        if (out_dt == BI8_F16) return by_layout(tag, static_cast<__half*>(nullptr));
        return by_layout(tag, static_cast<float*>(nullptr));
    };
    return s_dt == BI8_BF16 ? by_out(static_cast<__nv_bfloat16*>(nullptr)) : by_out(static_cast<__half*>(nullptr));
}

}  // namespace bi8
