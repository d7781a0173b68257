// Attention over a key/value cache that is held in 4-bit blocks of 64:
//   o[h, t] = sum_r p_r v_r,   p = softmax_r(scale * q[h, t] . k_r),   r from starts to the query's own row,
// with k_r = ks[r, j] / 7 * code and v_r the same.  The newest T rows of a sequence are its T queries (causal among them); heads of q
// share a head of the cache in groups of G = Hq / Hkv.  A query that sees no row gives zeros.
//
// What bounds one new token per sequence is the cache: D codes and D / 64 scales of k and of v for each row, read once for all G heads
// (0.53 bytes a value; at 6.5 TB/s 12 values per ns, three instructions of the SMs for each).  So the products are the tensor cores',
// with the codes as the 16-row operand of both (unpacked by one instruction a value, int4_common.cuh) and the queries, G * T of
// them, the eight columns:
//   S[row, query]  = sum_d k[row, d] q[query, d]
//   O[d, query]    = sum_row v[row, d] P[row, query]  two rows' words interleaved by byte permutes
// v's scales differ by row, so they go into P: p * vs as a sum of two fp16 numbers (22 bits), normalised by a power of two that
// follows the largest scale met, like the running maximum of the softmax.  P leaves the first product with its rows along the lanes and
// enters the second transposed (movmatrix).  Sums, statistics and scales are fp32.
//
// A warp takes steps of 16, 32 or 64 rows (4 KB) with the next step's loads in flight, straight into the registers that the matrix
// instructions read: no shared memory for the cache.  The warps of a CTA and the CTAs of a cluster divide the rows of one cache head
// (each reads the lengths and takes its share of what there really is) and are joined over distributed shared memory; more than eight
// shares go through a workspace and a second kernel.  Every sum has a fixed order.
#include "int4_common.cuh"

#include <cooperative_groups.h>

#include <type_traits>

namespace bi8 {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kClusterShares = 8;        // shares that a cluster joins
constexpr int kMaxShares = 64;

struct AttnArgs {
    const void* q;
    int64_t q_batch, q_head, q_tok;
    bi8_int4_cache cache;
    const long long* lengths;
    const long long* starts;
    int64_t lengths_step, starts_step;
    void* out;
    float* ws;               // [tile][share][8 NT][D] sums, then [tile][share][8 NT] pairs (maximum, total)
    int B, Hq, Hkv, T, G;
    int col_tiles, shares;
    float scale_log2;        // scale * log2(e)
};

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

// the scales of one row: U 16-bit values
template <int U>
struct RowScales {
    uint32_t w[(U + 1) / 2];
    __device__ __forceinline__ void load(const unsigned short* p) {
        if (U == 1) w[0] = __ldg(p);
        else if (U == 2) w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
        else {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
            w[0] = v.x;
            w[(U + 1) / 2 - 1] = v.y;
        }
    }
    template <typename T>
    __device__ __forceinline__ float get(int u) const { return u & 1 ? F16Bits<T>::hi(w[u / 2]) : F16Bits<T>::lo(w[u / 2]); }
};

template <int U, int TT>
struct Step {
    uint2 k[TT][2][U];           // rows g and g + 8 of each 16: eight bytes of every 64 values
    uint32_t v[TT][4][U];        // rows 2c, 2c + 1, 2c + 8, 2c + 9: four bytes of every 64 values
    RowScales<U> ks[TT][2], vs[TT][2];
};

template <int D>
constexpr int kStepTiles = D == 64 ? 4 : D == 128 ? 2 : 1;       // 16 rows each

template <int D, int NT>
constexpr int attn_smem() {
    // queries, the warps' sums (eight columns at a time), the CTA's sums, statistics
    return 8 * NT * (2 * D + 16) + kWarps * 8 * (D + 4) * 4 + 8 * NT * D * 4 + (kWarps * 2 + 2 + kClusterShares) * 8 * NT * 4 +
           8 * NT * 4;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads) attention_int4_kernel(const AttnArgs a) {
    constexpr int U = D / 64, TT = kStepTiles<D>, STEP = 16 * TT, COLS = 8 * NT, PITCH = 2 * D + 16, BUF = D + 4;
    extern __shared__ __align__(16) uint8_t smem[];
    uint8_t* const xs = smem;                                                    // [COLS] rows of PITCH bytes
    float* const buf = reinterpret_cast<float*>(xs + COLS * PITCH);              // [kWarps][8][BUF]
    float* const sums = buf + kWarps * 8 * BUF;                                  // [COLS][D]
    float* const warp_m = sums + COLS * D;                                       // [kWarps][COLS]
    float* const warp_l = warp_m + kWarps * COLS;                                // [kWarps][COLS]
    float* const cta_m = warp_l + kWarps * COLS;                                 // [COLS]
    float* const cta_l = cta_m + COLS;                                           // [COLS]
    float* const weight = cta_l + COLS;                                          // [kClusterShares][COLS]
    float* const factor = weight + kClusterShares * COLS;                        // [COLS]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int share = blockIdx.x % a.shares, tile = blockIdx.x / a.shares;
    const int ct = tile % a.col_tiles, bh = tile / a.col_tiles, h = bh % a.Hkv, b = bh / a.Hkv;
    const int R = a.G * a.T, col0 = ct * COLS, cols = min(COLS, R - col0);
    after_predecessor();

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
        *reinterpret_cast<uint4*>(xs + col * PITCH + p * 16) = operand8<T>(v, f.y);
        if (p == 0) factor[col] = a.scale_log2 * f.x * (1.0f / 7.0f);
    }
    __syncthreads();

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
    const int n_rows = max(0, most - start);
    const int chunk = (n_rows + a.shares * STEP - 1) / (a.shares * STEP) * STEP;
    const int first = start + min(n_rows, share * chunk), last = min(most, first + chunk);
    int limit[NT][2];
    float m[NT][2], l[NT][2], fac[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int col = 8 * t + 2 * c + j;
            limit[t][j] = col < cols ? min(last, rows_seen((col0 + col) % a.T)) : last;
            m[t][j] = -INFINITY;
            l[t][j] = 0.0f;
            fac[t][j] = factor[col];
        }
    const int unmasked = min(last, fewest);
    float o[NT][4 * U][4] = {};
    float vmax = 0x1p-110f;                               // power of two, no smaller than the scales of v so far (up to 2^127)

    const uint8_t* const kp = a.cache.k + b * a.cache.k_batch + h * a.cache.k_head + 8 * c;
    const uint8_t* const vp = a.cache.v + b * a.cache.v_batch + h * a.cache.v_head + 4 * g;
    const unsigned short* const ksp = static_cast<const unsigned short*>(a.cache.k_state) + b * a.cache.ks_batch + h * a.cache.ks_head;
    const unsigned short* const vsp = static_cast<const unsigned short*>(a.cache.v_state) + b * a.cache.vs_batch + h * a.cache.vs_head;
    auto load = [&](Step<U, TT>& s, int base) {           // rows behind the last one read that one again; they are masked
#pragma unroll
        for (int i = 0; i < TT; ++i) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int64_t row = min(base + 16 * i + g + 8 * r, last - 1);
#pragma unroll
                for (int u = 0; u < U; ++u) s.k[i][r][u] = __ldg(reinterpret_cast<const uint2*>(kp + row * (D / 2) + 32 * u));
                s.ks[i][r].load(ksp + row * U);
                s.vs[i][r].load(vsp + row * U);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t row = min(base + 16 * i + 2 * c + (r & 1) + 8 * (r >> 1), last - 1);
#pragma unroll
                for (int u = 0; u < U; ++u) s.v[i][r][u] = __ldg(reinterpret_cast<const uint32_t*>(vp + row * (D / 2) + 32 * u));
            }
        }
    };

    auto multiply = [&](const Step<U, TT>& s, int base, auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        // ---- scores
        float p[TT][NT][4] = {};
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint4* x = reinterpret_cast<const uint4*>(xs + (8 * t + g) * PITCH + u * 128 + c * 32);
                const uint4 xa = x[0], xb = x[1];
#pragma unroll
                for (int i = 0; i < TT; ++i) {
                    const Codes4 r0a = unpack8(s.k[i][0][u].x), r0b = unpack8(s.k[i][0][u].y);
                    const Codes4 r1a = unpack8(s.k[i][1][u].x), r1b = unpack8(s.k[i][1][u].y);
                    float d[4] = {};
                    mma_f16(d, r0a.p04, r1a.p04, r0a.p15, r1a.p15, xa.x, xa.y);
                    mma_f16(d, r0a.p26, r1a.p26, r0a.p37, r1a.p37, xa.z, xa.w);
                    mma_f16(d, r0b.p04, r1b.p04, r0b.p15, r1b.p15, xb.x, xb.y);
                    mma_f16(d, r0b.p26, r1b.p26, r0b.p37, r1b.p37, xb.z, xb.w);
                    const float s0 = s.ks[i][0].template get<T>(u), s1 = s.ks[i][1].template get<T>(u);
                    p[i][t][0] = fmaf(d[0], s0, p[i][t][0]);
                    p[i][t][1] = fmaf(d[1], s0, p[i][t][1]);
                    p[i][t][2] = fmaf(d[2], s1, p[i][t][2]);
                    p[i][t][3] = fmaf(d[3], s1, p[i][t][3]);
                }
            }
        // ---- softmax: running maximum and sum of every column
        bool grown = false;
        float alpha[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < TT; ++i)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float& x = p[i][t][2 * r + j];
                        x *= fac[t][j];
                        if (MASKED && base + 16 * i + g + 8 * r >= limit[t][j]) x = -INFINITY;
                        top = fmaxf(top, x);
                    }
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float now = fmaxf(m[t][j], top);
                const float ref = MASKED && now == -INFINITY ? 0.0f : now;      // a column that has seen nothing yet
                alpha[t][j] = exp2_fast(m[t][j] - ref);
                grown = grown || now != m[t][j];
                m[t][j] = now;
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < TT; ++i)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float& x = p[i][t][2 * r + j];
                        x = exp2_fast(x - ref);
                        sum += x;
                    }
                l[t][j] = fmaf(l[t][j], alpha[t][j], sum);
            }
        // ---- v's scales: a larger one than any before moves the normalisation
        float vs[TT][2][U], big = 0.0f;
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    vs[i][r][u] = s.vs[i][r].template get<T>(u);
                    big = fmaxf(big, vs[i][r][u]);
                }
        float shrink = 1.0f;
        if (__any_sync(0xffffffffu, big > vmax && vmax < 0x1p127f)) {
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
            const uint32_t e = min((__float_as_uint(big) >> 23) + 1u, 254u);
            const float next = __uint_as_float(e << 23);
            shrink = vmax / next;
            vmax = next;
            grown = true;
        }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int w = 0; w < 4 * U; ++w)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[t][w][j] *= alpha[t][j & 1] * shrink;
        }
        const float vscale = 0x1p14f / vmax;
        // ---- O += V^T P
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float s0 = vs[i][0][u] * vscale, s1 = vs[i][1][u] * vscale;
                uint32_t bh[NT][2], bl[NT][2];
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float sc = r ? s1 : s0;
                        float x0 = p[i][t][2 * r] * sc, x1 = p[i][t][2 * r + 1] * sc;
                        if (MASKED) {                     // a masked row's scale may be anything
                            const int row = base + 16 * i + g + 8 * r;
                            if (row >= limit[t][0]) x0 = 0.0f;
                            if (row >= limit[t][1]) x1 = 0.0f;
                        }
                        const uint32_t hi = pack_f16x2(x0, x1);
                        using H = F16Bits<__half>;
                        bh[t][r] = transpose8x8(hi);
                        bl[t][r] = transpose8x8(pack_f16x2(x0 - H::lo(hi), x1 - H::hi(hi)));
                    }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    // four codes of two rows: nibble n of both in bits 4n and 16 + 4n
                    const uint32_t w01 = __byte_perm(s.v[i][0][u], s.v[i][1][u], half ? 0x7632 : 0x5410);
                    const uint32_t w23 = __byte_perm(s.v[i][2][u], s.v[i][3][u], half ? 0x7632 : 0x5410);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t x = w01 >> (8 * j), y = w23 >> (8 * j);
                        const uint32_t a0 = codes_low(x), a1 = codes_high(x), a2 = codes_low(y), a3 = codes_high(y);
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            mma_f16(o[t][4 * u + 2 * half + j], a0, a1, a2, a3, bh[t][0], bh[t][1]);
                            mma_f16(o[t][4 * u + 2 * half + j], a0, a1, a2, a3, bl[t][0], bl[t][1]);
                        }
                    }
                }
            }
    };

    {
        Step<U, TT> cur, nxt;
        int base = first + warp * STEP;
        if (base < last) load(cur, base);
        for (; base < last; base += kWarps * STEP) {
            if (base + kWarps * STEP < last) load(nxt, base + kWarps * STEP);
            if (base + STEP <= unmasked) multiply(cur, base, std::false_type{});
            else multiply(cur, base, std::true_type{});
            cur = nxt;
        }
    }

    // ---- the warps' results into one
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[t][j] += __shfl_xor_sync(0xffffffffu, l[t][j], d);
            if (g == 0) {
                warp_m[warp * COLS + 8 * t + 2 * c + j] = m[t][j];
                warp_l[warp * COLS + 8 * t + 2 * c + j] = l[t][j];
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
    const float unit = vmax * (0x1p-14f / 7.0f);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int col = 2 * c + j;
            const float w = m[t][j] == -INFINITY ? 0.0f : exp2_fast(m[t][j] - cta_m[8 * t + col]) * unit;
            float* dst = buf + (warp * 8 + col) * BUF + 8 * g;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float x = w, y = w * 0.0625f;                  // the odd ones are 16 times too large
                *reinterpret_cast<float4*>(dst + 64 * u) = make_float4(o[t][4 * u][j] * x, o[t][4 * u][2 + j] * y, o[t][4 * u + 1][j] * x, o[t][4 * u + 1][2 + j] * y);
                *reinterpret_cast<float4*>(dst + 64 * u + 4) =
                    make_float4(o[t][4 * u + 2][j] * x, o[t][4 * u + 2][2 + j] * y, o[t][4 * u + 3][j] * x, o[t][4 * u + 3][2 + j] * y);
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 8 * D; i += kThreads) {
            const int col = i / D, d = i % D;
            float s = buf[col * BUF + d];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) s += buf[(w * 8 + col) * BUF + d];
            sums[(8 * t + col) * D + d] = s;
        }
        __syncthreads();
    }

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
        for (int r = 0; r < a.shares; ++r) {
            const float w = weight[r * COLS + col];
            const float2 v = *reinterpret_cast<const float2*>(cluster.map_shared_rank(sums, r) + col * D + d);
            x = fmaf(v.x, w, x);
            y = fmaf(v.y, w, y);
        }
        store(col, d, x, y);
    }
    cluster.sync();                                       // the others read this CTA's sums
}

// Joins the shares of one query: a CTA of D threads.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(D) attention_int4_join_kernel(const AttnArgs a, int64_t ctas) {
    constexpr int COLS = 8 * NT;
    __shared__ float weight[kMaxShares];
    after_predecessor();
    const int R = a.G * a.T, r = blockIdx.x % R, bh = blockIdx.x / R, h = bh % a.Hkv, b = bh / a.Hkv;
    const int64_t cta0 = ((int64_t)bh * a.col_tiles + r / COLS) * a.shares;
    const int col = r % COLS;
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
    const float* src = a.ws + (cta0 * COLS + col) * D + threadIdx.x;
    float x = 0.0f;
    for (int k = 0; k < a.shares; ++k) x = fmaf(src[(int64_t)k * COLS * D], weight[k], x);
    const int64_t at = (((int64_t)b * a.Hq + h * a.G + r / a.T) * a.T + r % a.T) * D + threadIdx.x;
    static_cast<unsigned short*>(a.out)[at] = (unsigned short)F16Bits<T>::pack(x, 0.0f);
}

int sm_count() {
    static int sms[64] = {0};
    int dev = 0;
    if (current_device(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (sms[dev] == 0) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) n = 148;
        sms[dev] = n;
    }
    return sms[dev];
}

struct Plan {
    int nt, col_tiles, shares;
    int64_t tiles;
};
Plan plan_of(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_len) {
    const int64_t R = Hq / Hkv * T;
    Plan p;
    p.nt = R <= 8 ? 1 : R <= 16 || D == 256 ? 2 : 4;
    p.col_tiles = (int)((R + 8 * p.nt - 1) / (8 * p.nt));
    p.tiles = B * Hkv * p.col_tiles;
    // Three CTAs an SM, as long as a warp of a full cache has two steps; the clusters' sizes are powers of two.
    const int64_t step = 16 * (D == 64 ? kStepTiles<64> : D == 128 ? kStepTiles<128> : kStepTiles<256>);
    const int64_t useful = (max_len + 2 * kWarps * step - 1) / (2 * kWarps * step), want = (3 * sm_count() + p.tiles - 1) / p.tiles;
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

template <typename T, int D, int NT>
int launch(const AttnArgs& a, int64_t tiles, cudaStream_t st) {
    constexpr int smem = attn_smem<D, NT>();
    static SmemOptIn opt_in;
    if (int rc = opt_in.ensure(attention_int4_kernel<T, D, NT>, smem)) return rc;
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
    BI8_CUDA_TRY(cudaLaunchKernelEx(&cfg, attention_int4_kernel<T, D, NT>, a));
    if (a.shares <= kClusterShares) return BI8_OK;
    return launch_chained(attention_int4_join_kernel<T, D, NT>, (unsigned)((int64_t)a.B * a.Hq * a.T), D, 0, st, a, (int64_t)grid);
}

}  // namespace

size_t attention_int4_workspace_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_len) {
    const Plan p = plan_of(B, T, Hq, Hkv, D, max_len);
    if (p.shares <= kClusterShares) return 0;
    return (size_t)(p.tiles * p.shares) * 8 * p.nt * (D + 2) * 4;
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
    a.scale_log2 = scale * 1.4426950408889634f;
    auto go = [&](auto* tag) {
        using E = std::remove_pointer_t<decltype(tag)>;
        if (D == 64) return p.nt == 1 ? launch<E, 64, 1>(a, p.tiles, st) : p.nt == 2 ? launch<E, 64, 2>(a, p.tiles, st) : launch<E, 64, 4>(a, p.tiles, st);
        if (D == 128) return p.nt == 1 ? launch<E, 128, 1>(a, p.tiles, st) : p.nt == 2 ? launch<E, 128, 2>(a, p.tiles, st) : launch<E, 128, 4>(a, p.tiles, st);
        return p.nt == 1 ? launch<E, 256, 1>(a, p.tiles, st) : launch<E, 256, 2>(a, p.tiles, st);
    };
    return dt == BI8_BF16 ? go(static_cast<__nv_bfloat16*>(nullptr)) : go(static_cast<__half*>(nullptr));
}

}  // namespace bi8
