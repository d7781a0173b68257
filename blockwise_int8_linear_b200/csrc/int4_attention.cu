// Attention over a key/value cache that is held in 4-bit blocks of 64:
//   o[h, t] = sum_r p_r v_r,   p = softmax_r(scale * q[h, t] . k_r),   r from starts to the query's own row,
// with k_r = ks[r, j] / 7 * code and v_r the same.  The newest T rows of a sequence are its T queries (causal among them); heads of q
// share a head of the cache in groups of G = Hq / Hkv.  A query that sees no row gives zeros.
//
// What bounds one new token per sequence is the cache: D codes and D / 64 scales of k and of v for each row, read once for all G heads
// (0.53 bytes a value; at 6.5 TB/s 12 values per ns, three instructions of the SMs for each).  So the products are the tensor cores',
// with the codes as the 16-row operand of both (unpacked by one instruction a value, int4_common.cuh) and the queries, G * T of
// them, eight at a time, the columns:
//   S[row, query]  = sum_d k[row, d] q[query, d]
//   O[d, query]    = sum_row v[row, d] P[row, query]  two rows' words interleaved by byte permutes
// v's scales differ by row, so they go into P: p * vs as a sum of two fp16 numbers (22 bits: one alone, 11 bits, is 9 % faster over long caches,
// but its roundings do not cancel where the values do, and leave a difference of nearly equal weights with two or three bits),
// normalised by a power of two that follows the largest p * vs that the query has met, like the running maximum of the softmax: a
// query's own, so that rows which it does not see have no part in its result, and of the products, so that large values of no weight
// take no bits from the others.  P leaves the first product with its rows along the lanes and enters the second transposed (movmatrix).
// Sums, statistics and scales are fp32.
//
// What bounds long caches: 815 instructions a step of 32 rows of 128 values, at an IPC of 2.4 of 4 (with 3.5 warps a scheduler, waits for the
// instruction before and for the integer pipe take the rest): 127000 rows of 8 heads in 45.5 us, 3.0 TB/s.  Short ones are latency: 4 us for the
// smallest call, 0.75 us a step.
//
// A warp takes steps of 16, 32 or 64 rows (4 KB), the next one on its way into shared memory while one is multiplied.  The warps of a CTA
// and the CTAs of a cluster divide the rows of one cache head (each reads the lengths and takes its share of what there really is) and
// are joined over distributed shared memory; more than eight shares go through a workspace and a second kernel.  Every sum has a
// fixed order.
#include "int4_common.cuh"

#include <cooperative_groups.h>

#include <type_traits>

namespace bi8 {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kCols = 8;                 // queries of a CTA
constexpr int kClusterShares = 8;        // shares that a cluster joins
constexpr int kMaxShares = 128;

struct AttnArgs {
    const void* q;
    int64_t q_batch, q_head, q_tok;
    bi8_int4_cache cache;
    const long long* lengths;
    const long long* starts;
    int64_t lengths_step, starts_step;
    void* out;
    float* ws;               // [tile][share][kCols][D] sums, then [tile][share][kCols] pairs (maximum, total)
    int B, Hq, Hkv, T, G;
    int col_tiles, shares;
    float scale_log2;        // scale * log2(e)
    bool s_vec;              // pairs of scales begin on 4-byte boundaries
};

// 2^e with |x| < 2^15 for x = max / 2^e (m: the bits of max in T), as the pair (2^e, 2^-e): what fits queries to fp16, which keeps
// everything of a bf16 value that is 2^-28 or more of the largest one.  Infinities and NaN stay what they are.
template <typename T>
__device__ __forceinline__ float2 fit_fp16(uint32_t m) {
    if (m == 0u || m >= F16Bits<T>::kInf) return make_float2(1.0f, 1.0f);
    int e = max((int)(__float_as_uint(F16Bits<T>::one(m)) >> 23), 1) - 127 - 14;          // denormals have the exponent -126
    e = max(e, -126 + 14);
    return make_float2(__uint_as_float((uint32_t)(e + 127) << 23), __uint_as_float((uint32_t)(127 - e) << 23));
}
template <typename T>
__device__ __forceinline__ uint4 scaled8(const uint4& v, float f) {
    using H = F16Bits<T>;
    return make_uint4(pack_f16x2(H::lo(v.x) * f, H::hi(v.x) * f), pack_f16x2(H::lo(v.y) * f, H::hi(v.y) * f), pack_f16x2(H::lo(v.z) * f, H::hi(v.z) * f),
                      pack_f16x2(H::lo(v.w) * f, H::hi(v.w) * f));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

template <int D>
constexpr int kStepTiles = D == 64 ? 4 : D == 128 ? 2 : 1;       // 16 rows each

template <int D>
constexpr int kResident = D == 256 ? 3 : 4;                     // CTAs of an SM

// A warp's rows of one step in shared memory: k, v, their scales.  A warp has two steps there: one in use, one on its way.
//
// Rows lie one behind the other without padding; the 16-byte pieces of every 128 bytes are permuted so that what the lanes read at a time
// lies in different banks: of k eight bytes (piece 2u + c / 2) of rows g, of v four bytes (piece 2u + g / 4) of every other row.  The
// permutation is an exclusive or with a number that is the same for rows eight apart, and so are its effects: a lane's address for the
// next 64 values or the next row is its first one with some bits flipped.
template <int D>
struct Ring {
    static constexpr int kRows = 16 * kStepTiles<D>, kRowScales = D / 64 * 2;
    static constexpr int kV = kRows * (D / 2), kScalesK = 2 * kV, kScalesV = kScalesK + kRows * kRowScales, kBytes = kScalesV + kRows * kRowScales;
    static constexpr int kSteps = 2;
    static __device__ __forceinline__ int at(int row, int piece) {
        if (D == 64) return (row >> 2) * 128 + ((((row & 3) << 1) | piece) ^ (((row >> 2) & 1) << 1)) * 16;
        if (D == 128) return (row >> 1) * 128 + ((((row & 1) << 2) | piece) ^ (((row >> 1) & 3) << 1)) * 16;
        return row * 128 + (piece ^ (((row ^ (row >> 1)) & 3) << 1)) * 16;
    }
    static constexpr int kOdd = D == 128 ? 64 : 32, kOddAdd = D == 256 ? 128 : 0;        // from an even row to the next: bits to flip, bytes to add
};

// Shared memory: queries; the warps' rings, afterwards the warps' sums and the CTA's; statistics.
template <int D>
struct Smem {
    static constexpr int kPitch = 2 * D + 16, kRings = kCols * kPitch, kBuf = D + 4;         // a query's row in bytes, a sum's in floats
    static constexpr int kRingBytes = kWarps * Ring<D>::kSteps * Ring<D>::kBytes, kSumBytes = (kWarps * kCols * kBuf + kCols * D) * 4;
    static constexpr int kStats = kRings + (kRingBytes > kSumBytes ? kRingBytes : kSumBytes);
    static constexpr int kBytes = kStats + (2 * kWarps + 3 + kClusterShares) * kCols * 4;
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, kResident<D>) attention_int4_kernel(const AttnArgs a) {
    constexpr int U = D / 64, TT = kStepTiles<D>, STEP = 16 * TT, COLS = kCols, PITCH = Smem<D>::kPitch, BUF = Smem<D>::kBuf;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* const xs = smem;                                                    // [COLS] rows of PITCH bytes
    uint8_t* const rings = smem + Smem<D>::kRings;                               // on a 128-byte boundary
    float* const warp_m = reinterpret_cast<float*>(smem + Smem<D>::kStats);      // [kWarps][COLS]
    float* const warp_l = warp_m + kWarps * COLS;                                // [kWarps][COLS]
    float* const cta_m = warp_l + kWarps * COLS;                                 // [COLS]
    float* const cta_l = cta_m + COLS;                                           // [COLS]
    float* const weight = cta_l + COLS;                                          // [kClusterShares][COLS]
    float* const factor = weight + kClusterShares * COLS;                        // [COLS]
    float* const buf = reinterpret_cast<float*>(rings);                          // [kWarps][8][BUF], when every warp has left its ring
    float* const sums = buf + kWarps * 8 * BUF;                                  // [COLS][D]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int share = blockIdx.x % a.shares, tile = blockIdx.x / a.shares;
    const int ct = tile % a.col_tiles, bh = tile / a.col_tiles, h = bh % a.Hkv, b = bh / a.Hkv;
    const int R = a.G * a.T, col0 = ct * COLS, cols = min(COLS, R - col0);
    after_predecessor();

    // ---- rows of this share
    const long long len = a.lengths[b * a.lengths_step];
    const int L = (int)a.cache.max_len;
    auto rows_seen = [&](int t) {                          // rows up to the query's own
        const long long n = len - a.T + t + 1;
        return (int)(n < 0 ? 0 : n > L ? L : n);
    };
    int start = 0;
    if (a.starts) {
        const long long s = a.starts[b * a.starts_step];
        start = (int)(s < 0 ? 0 : s > L ? L : s);
    }
    const bool one_head = col0 / a.T == (col0 + cols - 1) / a.T;
    const int fewest = rows_seen(one_head ? col0 % a.T : 0), most = rows_seen(one_head ? (col0 + cols - 1) % a.T : a.T - 1);
    // shares begin at multiples of 16 rows, which is what aligned copies of scales need; rows before `start` are masked
    const int origin = start & ~15, n_rows = most > start ? most - origin : 0;
    const int chunk = (n_rows + a.shares * STEP - 1) / (a.shares * STEP) * STEP;
    const int first = origin + min(n_rows, share * chunk), last = min(origin + n_rows, first + chunk);
    int limit[2];
    float m[2], l[2], fac[2];                              // running maximum (in powers of two) and total of a column, its factor
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int col = 2 * c + j;
        limit[j] = col < cols ? min(last, rows_seen((col0 + col) % a.T)) : last;
        m[j] = -INFINITY;
        l[j] = 0.0f;
    }
    const int unmasked = min(last, fewest);
    float o[4 * U][4] = {};
    float vtop[2] = {0.0f, 0.0f}, vmax[2] = {0x1p-110f, 0x1p-110f};      // a column's largest p * vs, and a power of two that is no smaller (2^127 at most)
    auto over = [](float pow2) { return __uint_as_float(((127u + 14u + 127u) << 23) - __float_as_uint(pow2)); };      // 2^14 / pow2

    const uint8_t* const kp = a.cache.k + b * a.cache.k_batch + h * a.cache.k_head;
    const uint8_t* const vp = a.cache.v + b * a.cache.v_batch + h * a.cache.v_head;
    const unsigned short* const ksp = static_cast<const unsigned short*>(a.cache.k_state) + b * a.cache.ks_batch + h * a.cache.ks_head;
    const unsigned short* const vsp = static_cast<const unsigned short*>(a.cache.v_state) + b * a.cache.vs_batch + h * a.cache.vs_head;
    using Slot = Ring<D>;
    uint8_t* const ring = rings + warp * (Slot::kSteps * Slot::kBytes);
    const int at_k = Slot::at(g, c >> 1) + 8 * (c & 1), at_v = Slot::at(2 * c, g >> 2) + 4 * (g & 3);       // this lane's first codes
    // One step's rows into a slot.  Rows behind the last one are that one again; they are masked.
    auto fill = [&](uint8_t* slot, int base) {
        constexpr int CH = D / 32;                         // 16-byte pieces of a row; 32 lanes take 32 / CH rows at a time
        const bool whole = base + STEP <= last;
        const int row0 = lane / CH, piece = lane % CH * 16;
        constexpr int AT_ONCE = 32 / CH;
        const uint32_t to = (uint32_t)__cvta_generic_to_shared(slot) + Slot::at(row0, lane % CH);
        const uint8_t *from_k = kp + (int64_t)base * (D / 2) + piece, *from_v = vp + (int64_t)base * (D / 2) + piece;
#pragma unroll
        for (int i = 0; i < STEP / AT_ONCE; ++i) {
            const int row = whole ? row0 + i * AT_ONCE : min(row0 + i * AT_ONCE, last - 1 - base);
            // rows that are not eight apart are permuted differently
            const uint32_t dst = AT_ONCE % 8 == 0 ? to + i * AT_ONCE * (D / 2) : (uint32_t)__cvta_generic_to_shared(slot) + Slot::at(row0 + i * AT_ONCE, lane % CH);
            copy16(dst, from_k + row * (D / 2));
            copy16(dst + Slot::kV, from_v + row * (D / 2));
        }
        if (U >= 2 || (a.s_vec && whole)) {                // a row's scales (two rows' where they have one) per lane, k and v in turn
            constexpr int BYTES = U == 4 ? 8 : 4, ROWS = BYTES / (2 * U), LANES = STEP / ROWS;
#pragma unroll
            for (int i = lane; i < 2 * LANES; i += 32) {
                const bool key = i < LANES;
                const int r = (key ? i : i - LANES) * ROWS, row = whole ? r : min(r, last - 1 - base);
                copy_some<BYTES>((uint32_t)__cvta_generic_to_shared(slot + (key ? Slot::kScalesK : Slot::kScalesV) + r * (2 * U)),
                                 (key ? ksp : vsp) + (int64_t)(base + row) * U);
            }
        } else {
            for (int r = lane; r < STEP; r += 32) {
                const int64_t row = min(base + r, last - 1);
                reinterpret_cast<unsigned short*>(slot + Slot::kScalesK)[r] = __ldg(ksp + row);
                reinterpret_cast<unsigned short*>(slot + Slot::kScalesV)[r] = __ldg(vsp + row);
            }
        }
    };
    // the scales of a row as floats
    auto scales_of = [&](const uint8_t* at, int row, float (&out)[U]) {
        if (U == 1) out[0] = F16Bits<T>::one(reinterpret_cast<const unsigned short*>(at)[row]);
#pragma unroll
        for (int i = 0; i < U / 2; ++i) {
            const uint32_t w = reinterpret_cast<const uint32_t*>(at)[row * (U / 2) + i];
            out[2 * i] = F16Bits<T>::lo(w);
            out[(2 * i + 1) % U] = F16Bits<T>::hi(w);
        }
    };

    auto multiply = [&](const uint8_t* slot, int base, auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        // ---- scores
        float p[TT][4] = {};
#pragma unroll
        for (int i = 0; i < TT; ++i) {
            float s0[U], s1[U];
            scales_of(slot + Slot::kScalesK, 16 * i + g, s0);
            scales_of(slot + Slot::kScalesK, 16 * i + g + 8, s1);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint8_t* const k = slot + (at_k ^ (32 * u)) + 16 * i * (D / 2);
                const uint2 w0 = *reinterpret_cast<const uint2*>(k), w1 = *reinterpret_cast<const uint2*>(k + 8 * (D / 2));
                const Codes4 r0a = unpack8<__half>(w0.x), r0b = unpack8<__half>(w0.y), r1a = unpack8<__half>(w1.x), r1b = unpack8<__half>(w1.y);
                const uint4* x = reinterpret_cast<const uint4*>(xs + g * PITCH + u * 128 + c * 32);
                const uint4 xa = x[0], xb = x[1];
                float d[4];
                mma16_first<__half>(d, r0a.p04, r1a.p04, r0a.p15, r1a.p15, xa.x, xa.y);
                mma16<__half>(d, r0a.p26, r1a.p26, r0a.p37, r1a.p37, xa.z, xa.w);
                mma16<__half>(d, r0b.p04, r1b.p04, r0b.p15, r1b.p15, xb.x, xb.y);
                mma16<__half>(d, r0b.p26, r1b.p26, r0b.p37, r1b.p37, xb.z, xb.w);
                p[i][0] = fmaf(d[0], s0[u], p[i][0]);
                p[i][1] = fmaf(d[1], s0[u], p[i][1]);
                p[i][2] = fmaf(d[2], s1[u], p[i][2]);
                p[i][3] = fmaf(d[3], s1[u], p[i][3]);
            }
        }
        // ---- softmax: running maximum and sum of every column
        bool grown = false;
        float alpha[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < TT; ++i)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float& x = p[i][2 * r + j];
                    x = __fmul_rn(x, fac[j]);             // the column's factor is not negative
                    if (MASKED && (base + 16 * i + g + 8 * r >= limit[j] || base + 16 * i + g + 8 * r < start)) x = -INFINITY;
                    top = fmaxf(top, x);
                }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            // The running maximum is one of the rounded products that it is subtracted from.  So nothing is above it, however large the scores (the
            // product's rounding error alone may be: in one multiply-add of 1e20 it would be 2^40 to the exponential), and where it has not
            // grown, total and sums are rescaled by 1.  A column may have seen nothing yet.
            const float now = fmaxf(m[j], top), ref = now == -INFINITY ? 0.0f : now;
            alpha[j] = exp2_fast(m[j] - ref);
            grown = grown || now != m[j];
            m[j] = now;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < TT; ++i)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float& x = p[i][2 * r + j];
                    x = exp2_fast(x - ref);
                    sum += x;
                }
            l[j] = fmaf(l[j], alpha[j], sum);
        }
        // ---- times v's scales: a larger product than any before moves the column's normalisation
        float pv[TT][2][U][2], big[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float vs[U];
                scales_of(slot + Slot::kScalesV, 16 * i + g + 8 * r, vs);
                const int row = base + 16 * i + g + 8 * r;
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const bool unseen = MASKED && (row >= limit[j] || row < start);          // its scale may be anything
                        pv[i][r][u][j] = unseen ? 0.0f : p[i][2 * r + j] * vs[u];
                        big[j] = fmaxf(big[j], fabsf(pv[i][r][u][j]));                            // passes over the NaN of blocks that hold one
                    }
            }
        if (__any_sync(0xffffffffu, grown || big[0] > vmax[0] || big[1] > vmax[1])) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float top = big[j];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                vtop[j] = fmaxf(vtop[j] * alpha[j], top);
                const float next = __uint_as_float(min(max((__float_as_uint(vtop[j]) + 0x7fffffu) >> 23, 127u - 110u), 254u) << 23);
                alpha[j] = alpha[j] * vmax[j] * over(next) * 0x1p-14f;      // vmax is the smallest number, or below twice what vtop was: at most 2^15 on the way
                vmax[j] = next;
            }
#pragma unroll
            for (int w = 0; w < 4 * U; ++w)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[w][j] *= alpha[j & 1];
        }
        // ---- O += V^T P
        const float vscale[2] = {over(vmax[0]), over(vmax[1])};
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint32_t bh[2], bl[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float x0 = pv[i][r][u][0] * vscale[0], x1 = pv[i][r][u][1] * vscale[1];
                    const uint32_t hi = pack_f16x2(x0, x1);
                    using H = F16Bits<__half>;
                    bh[r] = transpose8x8(hi);
                    bl[r] = transpose8x8(pack_f16x2(x0 - H::lo(hi), x1 - H::hi(hi)));
                }
                const uint8_t* const even = slot + (at_v ^ (32 * u)) + Slot::kV + 16 * i * (D / 2);
                const uint8_t* const odd = slot + ((at_v ^ (32 * u)) ^ Slot::kOdd) + Slot::kOddAdd + Slot::kV + 16 * i * (D / 2);
                uint32_t w[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) w[r] = *reinterpret_cast<const uint32_t*>((r & 1 ? odd : even) + 8 * (r >> 1) * (D / 2));
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    // four codes of two rows: nibble n of both in bits 4n and 16 + 4n
                    const uint32_t w01 = __byte_perm(w[0], w[1], half ? 0x7632 : 0x5410);
                    const uint32_t w23 = __byte_perm(w[2], w[3], half ? 0x7632 : 0x5410);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t x = w01 >> (8 * j), y = w23 >> (8 * j);
                        const uint32_t a0 = half2_low(x), a1 = half2_high(x), a2 = half2_low(y), a3 = half2_high(y);
                        mma16<__half>(o[4 * u + 2 * half + j], a0, a1, a2, a3, bh[0], bh[1]);
                        mma16<__half>(o[4 * u + 2 * half + j], a0, a1, a2, a3, bl[0], bl[1]);
                    }
                }
            }
    };

    int in = 0, out = 0;                                  // slots of the ring
    auto fill_next = [&](int base) {
        if (base < last) fill(ring + in * Slot::kBytes, base);
        commit_copies();
        in = in + 1 == Slot::kSteps ? 0 : in + 1;
    };
#pragma unroll
    for (int i = 0; i < Slot::kSteps - 1; ++i) fill_next(first + (warp + i * kWarps) * STEP);

    // ---- queries: fp16 with a power of two per query; D / 8 lanes a query
    for (int i = threadIdx.x; i < COLS * (D / 8); i += kThreads) {
        const int col = i / (D / 8), p = i % (D / 8), r = col0 + col;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (col < cols)
            v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.q_batch + (int64_t)(h * a.G + r / a.T) * a.q_head + (r % a.T) * a.q_tok + 8 * p);
        uint32_t big = absmax8(v);
#pragma unroll
        for (int d = 1; d < D / 8; d <<= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, d));
        const float2 f = fit_fp16<T>(big);
        *reinterpret_cast<uint4*>(xs + col * PITCH + p * 16) = paired8(scaled8<T>(v, a.scale_log2 < 0.0f ? -f.y : a.scale_log2 > 0.0f ? f.y : 0.0f));
        // never 0, which the infinities of unseen rows do not bear (a scale of 0 makes the queries 0)
        if (p == 0) factor[col] = a.scale_log2 == 0.0f ? 1.0f : fmaxf(fabsf(a.scale_log2) * f.x * (1.0f / 7.0f), 0x1p-126f);
    }
    __syncthreads();

#pragma unroll
    for (int j = 0; j < 2; ++j) fac[j] = factor[2 * c + j];

    for (int base = first + warp * STEP; base < last; base += kWarps * STEP) {
        fill_next(base + (Slot::kSteps - 1) * kWarps * STEP);         // into the slot that every lane left at the end of the step before
        wait_copies<Slot::kSteps - 1>();
        __syncwarp();
        if (base >= start && base + STEP <= unmasked) multiply(ring + out * Slot::kBytes, base, std::false_type{});
        else multiply(ring + out * Slot::kBytes, base, std::true_type{});
        __syncwarp();
        out = out + 1 == Slot::kSteps ? 0 : out + 1;
    }
    wait_copies<0>();

    // ---- the warps' results into one
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], d);
        if (g == 0) {
            warp_m[warp * COLS + 2 * c + j] = m[j];
            warp_l[warp * COLS + 2 * c + j] = l[j];
        }
    }
    __syncthreads();
    for (int col = threadIdx.x; col < COLS; col += kThreads) {
        float top = -INFINITY, total = 0.0f;
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, warp_m[w * COLS + col]);
        for (int w = 0; w < kWarps; ++w)
            if (warp_l[w * COLS + col] != 0.0f) total += warp_l[w * COLS + col] * exp2_fast(warp_m[w * COLS + col] - top);
        cta_m[col] = top;
        cta_l[col] = total;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int col = 2 * c + j;
        const float w = m[j] == -INFINITY ? 0.0f : exp2_fast(m[j] - cta_m[col]) * (vmax[j] * (0x1p-14f / 7.0f));
        float* dst = buf + (warp * 8 + col) * BUF + 8 * g;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            *reinterpret_cast<float4*>(dst + 64 * u) = make_float4(o[4 * u][j] * w, o[4 * u][2 + j] * w, o[4 * u + 1][j] * w, o[4 * u + 1][2 + j] * w);
            *reinterpret_cast<float4*>(dst + 64 * u + 4) =
                make_float4(o[4 * u + 2][j] * w, o[4 * u + 2][2 + j] * w, o[4 * u + 3][j] * w, o[4 * u + 3][2 + j] * w);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * D; i += kThreads) {
        const int col = i / D, d = i % D;
        float s = buf[col * BUF + d];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) s += buf[(w * 8 + col) * BUF + d];
        sums[col * D + d] = s;
    }
    __syncthreads();

    auto store = [&](int col, int d, float x, float y) {
        const int r = col0 + col;
        const int64_t at = (((int64_t)b * a.Hq + h * a.G + r / a.T) * a.T + r % a.T) * D + d;
        *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + at) = F16Bits<T>::pack(x, y);
    };
    if (a.shares == 1) {
        for (int i = threadIdx.x; i < cols * (D / 2); i += kThreads) {
            const int col = i / (D / 2), d = i % (D / 2) * 2;
            const float total = cta_l[col], inv = total == 0.0f ? 0.0f : 1.0f / total;
            store(col, d, sums[col * D + d] * inv, sums[col * D + d + 1] * inv);
        }
        return;
    }
    if (a.shares > kClusterShares) {
        float* dst = a.ws + (int64_t)blockIdx.x * COLS * D;
        for (int i = threadIdx.x; i < cols * D; i += kThreads) dst[i] = sums[i];
        float2* stat = reinterpret_cast<float2*>(a.ws + (int64_t)gridDim.x * COLS * D) + (int64_t)blockIdx.x * COLS;
        for (int i = threadIdx.x; i < cols; i += kThreads) stat[i] = make_float2(cta_m[i], cta_l[i]);
        return;
    }
    const cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int col = threadIdx.x; col < cols; col += kThreads) {
        float ms[kClusterShares], ls[kClusterShares], top = -INFINITY, total = 0.0f;
#pragma unroll
        for (int r = 0; r < kClusterShares; ++r) {
            ms[r] = -INFINITY;
            ls[r] = 0.0f;
            if (r < a.shares) {
                ms[r] = cluster.map_shared_rank(cta_m, r)[col];
                ls[r] = cluster.map_shared_rank(cta_l, r)[col];
            }
            top = fmaxf(top, ms[r]);
        }
#pragma unroll
        for (int r = 0; r < kClusterShares; ++r) {
            ms[r] = ls[r] != 0.0f ? exp2_fast(ms[r] - top) : 0.0f;
            total += ls[r] * ms[r];
        }
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int r = 0; r < kClusterShares; ++r) weight[r * COLS + col] = ms[r] * inv;
    }
    __syncthreads();
    const int pairs = cols * (D / 2), part = (pairs + a.shares - 1) / a.shares;
    for (int i = share * part + threadIdx.x; i < min(pairs, (share + 1) * part); i += kThreads) {
        const int col = i / (D / 2), d = i % (D / 2) * 2;
        float x = 0.0f, y = 0.0f;
        float2 v[kClusterShares];
#pragma unroll
        for (int r = 0; r < kClusterShares; ++r)
            if (r < a.shares) v[r] = *reinterpret_cast<const float2*>(cluster.map_shared_rank(sums, r) + col * D + d);
#pragma unroll
        for (int r = 0; r < kClusterShares; ++r)
            if (r < a.shares) {
                x = fmaf(v[r].x, weight[r * COLS + col], x);
                y = fmaf(v[r].y, weight[r * COLS + col], y);
            }
        store(col, d, x, y);
    }
    cluster.sync();                                       // the others read this CTA's sums
}

// Joins the shares of one query: a CTA of four times D threads, a quarter of the shares each.
template <typename T, int D>
__global__ void __launch_bounds__(4 * D) attention_int4_join_kernel(const AttnArgs a, int64_t ctas) {
    constexpr int COLS = kCols;
    __shared__ float weight[kMaxShares];
    __shared__ float sum[4][D];
    after_predecessor();
    const int R = a.G * a.T, r = blockIdx.x % R, bh = blockIdx.x / R, h = bh % a.Hkv, b = bh / a.Hkv;
    const int64_t cta0 = ((int64_t)bh * a.col_tiles + r / COLS) * a.shares;
    const int col = r % COLS, d = threadIdx.x % D, part = threadIdx.x / D;
    const int per = (a.shares + 3) / 4, first = part * per, last = min(a.shares, first + per);
    const float* src = a.ws + (cta0 * COLS + col) * D + d;
    float v[8];                                           // on their way before the weights are known
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = first + k < last ? src[(int64_t)(first + k) * COLS * D] : 0.0f;
    const float2* stat = reinterpret_cast<const float2*>(a.ws + ctas * COLS * D) + cta0 * COLS + col;
    if (threadIdx.x < 32) {
        float top = -INFINITY, total = 0.0f;
        float2 s[kMaxShares / 32];
#pragma unroll
        for (int i = 0; i < kMaxShares / 32; ++i) {
            const int k = threadIdx.x + 32 * i;
            s[i] = k < a.shares ? stat[(int64_t)k * COLS] : make_float2(-INFINITY, 0.0f);
            top = fmaxf(top, s[i].x);
        }
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
#pragma unroll
        for (int i = 0; i < kMaxShares / 32; ++i) {
            s[i].x = s[i].y != 0.0f ? exp2_fast(s[i].x - top) : 0.0f;
            total += s[i].x * s[i].y;
        }
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int i = 0; i < kMaxShares / 32; ++i) weight[threadIdx.x + 32 * i] = s[i].x * inv;
    }
    __syncthreads();
    float x = 0.0f;
    for (int k0 = first; k0 < last; k0 += 8) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k0 + k < last) x = fmaf(v[k], weight[k0 + k], x);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = k0 + 8 + k < last ? src[(int64_t)(k0 + 8 + k) * COLS * D] : 0.0f;
    }
    sum[part][d] = x;
    __syncthreads();
    if (part > 0) return;
    const int64_t at = (((int64_t)b * a.Hq + h * a.G + r / a.T) * a.T + r % a.T) * D + d;
    static_cast<unsigned short*>(a.out)[at] = (unsigned short)F16Bits<T>::pack((sum[0][d] + sum[1][d]) + (sum[2][d] + sum[3][d]), 0.0f);
}

struct Plan {
    int col_tiles, shares;
    int64_t tiles;
};
Plan plan_of(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_len) {
    const int64_t R = Hq / Hkv * T;
    Plan p;
    p.col_tiles = (int)((R + kCols - 1) / kCols);
    p.tiles = B * Hkv * p.col_tiles;
    // As many CTAs as the device holds at once.  Few tiles are divided down to a step for each warp (one sequence of 2048 rows, 8 heads: 19 us in
    // 1 share, 8.6 in 4, 6.2 in 16), beyond two CTAs an SM into 512 rows and more (16384 rows: 14.2 us in 16 shares, 12.3 in 32, 13.9 in 74), more
    // tiles than SMs only into 1024 rows and more (256 tiles of 576 rows: 11.5 us in 1, 12.4 in 2).  Long
    // caches, whose sequences may differ much in length, have shares of 2048 rows (32 sequences of 1 to 8192 rows, 8 heads: 79 us in 2, 62
    // in 4, 66 in 8; 64 of 4096 rows each: 88 us in 1, 80 in 2, 92 in 4).  The clusters' sizes are powers of two.
    const int64_t step = 16 * (D == 64 ? kStepTiles<64> : D == 128 ? kStepTiles<128> : kStepTiles<256>), sms = sm_count();
    const int64_t useful = p.tiles < sms ? (max_len + kWarps * step - 1) / (kWarps * step) : max_len / 1024, long_ones = max_len / 2048;
    int64_t want = (D == 256 ? kResident<256> : kResident<128>) * sms / p.tiles;
    const int64_t two = 2 * sms / p.tiles, half = max_len / 512;
    if (want > two && want > half) want = two > half ? two : half;
    if (want < kClusterShares && want < long_ones) want = long_ones < kClusterShares ? long_ones : kClusterShares;
    int64_t s = useful < want ? useful : want;
    if (s > kMaxShares) s = kMaxShares;
    if (s <= kClusterShares) {
        int64_t pow = 1;
        while (pow * 2 <= s) pow *= 2;
        s = pow;
    }
    p.shares = (int)(s < 1 ? 1 : s);
    return p;
}

template <typename T, int D>
int launch(const AttnArgs& a, int64_t tiles, cudaStream_t st) {
    constexpr int smem = Smem<D>::kBytes;
    static SmemOptIn opt_in;
    if (int rc = opt_in.ensure(attention_int4_kernel<T, D>, smem)) return rc;
    const unsigned grid = (unsigned)(tiles * a.shares);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.shares <= kClusterShares ? (unsigned)a.shares : 1u;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    BI8_CUDA_TRY(cudaLaunchKernelEx(&cfg, attention_int4_kernel<T, D>, a));
    if (a.shares <= kClusterShares) return BI8_OK;
    return launch_chained(attention_int4_join_kernel<T, D>, (unsigned)((int64_t)a.B * a.Hq * a.T), 4 * D, 0, st, a, (int64_t)grid);
}

}  // namespace

size_t attention_int4_workspace_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_len) {
    const Plan p = plan_of(B, T, Hq, Hkv, D, max_len);
    if (p.shares <= kClusterShares) return 0;
    return (size_t)(p.tiles * p.shares) * kCols * (D + 2) * 4;
}

int launch_attention_int4(const void* q, int dt, int64_t q_batch, int64_t q_head, int64_t q_tok, const bi8_int4_cache* cache, const long long* lengths,
                          int64_t lengths_step, const long long* starts, int64_t starts_step, float scale, void* out, int64_t B, int64_t T, int64_t Hq,
                          int64_t Hkv, int64_t D, void* workspace, cudaStream_t st) {
    const Plan p = plan_of(B, T, Hq, Hkv, D, cache->max_len);
    if (p.tiles * p.shares > 0x7fffffff || B * Hq * T > 0x7fffffff)
        return fail(BI8_ERR_LIMIT, "attention_int4: %lld queries exceed one launch", (long long)(B * Hq * T));
    AttnArgs a{};
    a.q = q;
    a.q_batch = q_batch;
    a.q_head = q_head;
    a.q_tok = q_tok;
    a.cache = *cache;
    a.lengths = lengths;
    a.lengths_step = lengths_step;
    a.starts = starts;
    a.starts_step = starts_step;
    a.out = out;
    a.ws = static_cast<float*>(workspace);
    a.B = (int)B;
    a.Hq = (int)Hq;
    a.Hkv = (int)Hkv;
    a.T = (int)T;
    a.G = (int)(Hq / Hkv);
    a.col_tiles = p.col_tiles;
    a.shares = p.shares;
    a.s_vec = aligned(cache->k_state, 4) && aligned(cache->v_state, 4) && cache->ks_batch % 2 == 0 && cache->ks_head % 2 == 0 && cache->vs_batch % 2 == 0 &&
              cache->vs_head % 2 == 0;
    a.scale_log2 = scale * 1.4426950408889634f;
    auto go = [&](auto* tag) {
        using E = std::remove_pointer_t<decltype(tag)>;
        if (D == 64) return launch<E, 64>(a, p.tiles, st);
        if (D == 128) return launch<E, 128>(a, p.tiles, st);
        return launch<E, 256>(a, p.tiles, st);
    };
    return dt == BI8_BF16 ? go(static_cast<__nv_bfloat16*>(nullptr)) : go(static_cast<__half*>(nullptr));
}

}  // namespace bi8
