// Attention of a few queries of each cache head over a paged 16-bit cache:
//   o[q] = sum_r p_r v_r,   p = softmax_r(scale * q . k_r),   r from the sequence's start to the query's own row.
//
// The new tokens of a sequence are its last rows (causal among them); heads of q share a head of the cache in groups of G.  A query that sees no
// row gives zeros.
//
// What bounds it is the cache, 4 D bytes a row and head, read once for up to kCols queries.  So the products are the tensor cores' with the
// queries as the 16-row operand, whether or not there are 16 of them:
//   S[query, row] = sum_d q[query, d] k[row, d]      O[query, d] = sum_row P[query, row] v[row, d]
// S leaves the first product in the layout in which P enters the second.  P goes there as a sum of two 16-bit numbers: one alone would lose as
// much as the result's own rounding does, and the second product has time to spare.  Sums and statistics are fp32.
//
// A warp takes steps of 16 or 32 rows, kSlots - 1 of them on their way into shared memory while one is multiplied.  The warps of a CTA and the CTAs of
// a cluster divide the rows (each reads the lengths and takes its share of what there really is) and are joined over distributed shared
// memory; more than eight shares go through a workspace and a second kernel.  Every sum has a fixed order.
//
// One sequence of 131072 rows, 32 heads on 8: 87 to 90 us, 91 to 94 % of a copy's bandwidth; 32 sequences of 1 to 8192 rows: 101 to 111 us from one GPU to another, 76
// to 84 %, because a CTA's first rows come 2 to 3 us after the last ones of the CTA whose place it takes; 600 rows alone: 7.7 to 8.3 us, latency.  Heads of
// 256, 32 on 8: 8 sequences of 4000 rows 61 us (40 by the bytes), 32 of them 261 to 276 (160): one CTA an SM.
//
// Rows that a sequence does not have, or that come before its start, are not read: they are zeros in shared memory, so that whatever is in the
// cache there, infinities and NaN among it, has no part in the products.  Those of rows that only some of the queries see take a way of their own
// (paged_attention.cuh).
#include "paged_attention.cuh"

#include <cooperative_groups.h>

#include <cmath>
#include <type_traits>

namespace bi8 {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kCols = kFewQueries;       // queries of a CTA
constexpr int kClusterShares = 8, kMaxShares = 128;
constexpr int kSingleRound = 2;          // CTAs of an SM where more shares than a cluster's make one round of CTAs (few_shares): with a step more on its way in each warp

template <int D>
constexpr int kSubSteps = D == 64 ? 2 : 1;          // 16 rows each
template <int D>
constexpr int kResident = D == 256 ? 1 : 3;         // CTAs of an SM

// Shared memory: the warps' rings (k and v of a step in each slot), afterwards the warps' sums and the CTA's; queries; statistics.  The 16-byte
// pieces of a row are permuted by the row's number, so that the eight rows of a matrix lie in different banks.
template <int D, int kSlots>
struct Smem {
    static constexpr int kStep = 16 * kSubSteps<D>, kRow = 2 * D, kV = kStep * kRow, kSlot = 2 * kV;
    static constexpr int kBuf = D + 4;                                   // a sum's row in floats
    static constexpr int kRingBytes = kWarps * kSlots * kSlot, kSumBytes = (kWarps * kCols * kBuf + kCols * D) * 4;
    static constexpr int kQueries = kRingBytes > kSumBytes ? kRingBytes : kSumBytes;
    static constexpr int kStats = kQueries + kCols * kRow;
    static constexpr int kNoted = kStats + (2 * kWarps + 2 + kClusterShares) * kCols * 4, kBytes = kNoted + 16;
};

__device__ __forceinline__ void load_matrices(uint32_t at, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_matrices_transposed(uint32_t at, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

template <typename T, int D, int kSlots>
__global__ void __launch_bounds__(kThreads, kSlots == 3 ? kSingleRound : kResident<D>) paged_few_kernel(const PagedAttnArgs a) {
    using L = Smem<D, kSlots>;
    constexpr int TT = kSubSteps<D>, STEP = L::kStep, PIECES = D / 8, CHUNKS = D / 16, BUF = L::kBuf;
    extern __shared__ __align__(128) uint8_t smem[];
    float* const warp_m = reinterpret_cast<float*>(smem + L::kStats);            // [kWarps][kCols]
    float* const warp_l = warp_m + kWarps * kCols;                               // [kWarps][kCols]
    float* const cta_m = warp_l + kWarps * kCols;                                // [kCols]
    float* const cta_l = cta_m + kCols;                                          // [kCols]
    float* const weight = cta_l + kCols;                                         // [kClusterShares][kCols]
    float* const buf = reinterpret_cast<float*>(smem);                           // [kWarps][kCols][BUF], when every warp has left its ring
    float* const sums = buf + kWarps * kCols * BUF;                              // [kCols][D]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int tile_head = (int)a.per_share.div(blockIdx.x), share = (int)blockIdx.x - tile_head * a.shares;
    const int tile = (int)a.heads.div((unsigned)tile_head), h = tile_head - tile * a.Hkv;
    const Sequences& s = a.seq;
    QueryTile qt;
    if (a.by_length) {
        // Behind the kernel for many queries, which waits for what came before it when it begins: this one reads and writes nothing of that kernel's and
        // takes the SMs that it leaves.  Its first CTA waits for that kernel before it ends, so that whoever waits for this one has waited for both;
        // the others leave their places to the next.  Without a wait of its own it reads what earlier kernels wrote from the L2 (bi8_common.cuh): numbers and
        // queries by ld_l2, the cache by copies that pass by the SM's own.  (16 sequences of up to 4096 rows, one with 33 tokens: 101 us, 99 by ordinary loads.  A
        // fence in each CTA: 106.)
        const int first = s.first_token<true>(tile), n = max(s.first_token<true>(tile + 1) - first, 0);
        qt = {tile, n, first, 0, (int64_t)n * a.G <= kCols ? n * a.G : 0};
    } else {
        after_predecessor();
        qt = find_tile(s, tile, a.G, kCols, a.per_sequence);
    }
    if (qt.rows == 0) {                                                          // the whole cluster's tile
        if (a.by_length && blockIdx.x == 0) wait_predecessor();
        return;
    }
    auto token_of = [&](int r) { return (int)a.group.div((unsigned)(qt.row0 + r)); };

    // ---- queries, on their way while the rest is found out
    constexpr int Q_LOADS = kCols * PIECES / kThreads;
    const int q_piece = threadIdx.x % PIECES;
    uint4 query[Q_LOADS];
#pragma unroll
    for (int i = 0; i < Q_LOADS; ++i) {
        const int r = (int)threadIdx.x / PIECES + i * (kThreads / PIECES);
        query[i] = make_uint4(0u, 0u, 0u, 0u);
        if (r < qt.rows) {
            const int t = token_of(r), head = h * a.G + (qt.row0 + r - t * a.G);
            query[i] = ld_l2(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (int64_t)(qt.token0 + t) * a.q_tok + head * a.q_head + 8 * q_piece));
        }
    }

    // ---- rows of this share
    const long long position = s.first_position<true>(qt.b, qt.n);
    const int fewest = rows_seen(s, position, token_of(0)), most = rows_seen(s, position, token_of(qt.rows - 1));
    const int start = s.start<true>(qt.b), origin = start & ~15, n_rows = most > start ? most - origin : 0;
    const int chunk = (n_rows + a.shares * STEP - 1) / (a.shares * STEP) * STEP;
    const int first = origin + min(n_rows, share * chunk), last = min(origin + n_rows, first + chunk);
    int limit[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = g + 8 * i;
        limit[i] = r < qt.rows ? min(last, rows_seen(s, position, token_of(r))) : last;      // a query that is none sees all: it is zero
    }
    const int unmasked = min(last, fewest);
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};             // running maximum (in powers of two) and total of queries g and g + 8
    float o[D / 8][4] = {};

    // ---- the ring: a row's 16-byte pieces by as many lanes
    const int* const pages = s.pages + (qt.b < s.B ? qt.b : 0) * s.pages_step;
    const char* const kh = static_cast<const char*>(a.cache.k) + 2 * h * a.cache.k_head;
    const char* const vh = static_cast<const char*>(a.cache.v) + 2 * h * a.cache.v_head;
    const char* const nothing = static_cast<const char*>(a.q);                  // an address for copies of no bytes
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (kSlots * L::kSlot);
    constexpr int AT_ONCE = 32 / PIECES == 0 ? 1 : 32 / PIECES;                 // rows of a warp's access
    const int row0 = lane / PIECES, piece = lane % PIECES;
    constexpr int AHEAD = kWarps * STEP;
    struct Pages {
        int number[TT];
    };
    // elsewhere from the SM's own cache, since consecutive numbers lie together (8 sequences of 4000 rows, D 256: 68 us, 71 from the L2)
    auto page_number = [&](const int* p) { return a.by_length ? ld_l2(p) : *p; };
    auto pages_of = [&](int base) {
        Pages p;
#pragma unroll
        for (int i = 0; i < TT; ++i) p.number[i] = base + 16 * i < last ? page_number(pages + s.page.div((unsigned)(base + 16 * i))) : -1;
        return p;
    };
    auto fill = [&](uint32_t slot, int base, const Pages& p) {
#pragma unroll
        for (int i = 0; i < TT; ++i) {
            const int sub = base + 16 * i, in_page = sub - (int)s.page.div((unsigned)sub) * (int)s.page.d;
            const bool there = p.number[i] >= 0 && p.number[i] < a.cache.pages;
            const int64_t page = there ? p.number[i] : 0;
            const char* const from_k = kh + 2 * (page * a.cache.k_page + (in_page + row0) * a.cache.k_row) + 16 * piece;
            const char* const from_v = vh + 2 * (page * a.cache.v_page + (in_page + row0) * a.cache.v_row) + 16 * piece;
#pragma unroll
            for (int j = 0; j < 16 / AT_ONCE; ++j) {
                const int r = row0 + j * AT_ONCE, row = sub + r;
                const int bytes = there && row >= start && row < last ? 16 : 0;
                const uint32_t to = slot + (16 * i + r) * L::kRow + 16 * (piece ^ (r & 7));
                copy16(to, bytes ? from_k + 2 * j * AT_ONCE * a.cache.k_row : nothing, bytes);
                copy16(to + L::kV, bytes ? from_v + 2 * j * AT_ONCE * a.cache.v_row : nothing, bytes);
            }
        }
    };

    unsigned* const noted = reinterpret_cast<unsigned*>(smem + L::kNoted);      // rows from `fewest` on with values that are not finite
    if (threadIdx.x == 0) *noted = 0u;
    const uint32_t queries = (uint32_t)__cvta_generic_to_shared(smem + L::kQueries);
    int base = first + warp * STEP;
#pragma unroll
    for (int i = 0; i < kSlots - 1; ++i) {
        if (base + i * AHEAD < last) fill(ring + i * L::kSlot, base + i * AHEAD, pages_of(base + i * AHEAD));
        commit_copies();
    }
    Pages next = pages_of(base + (kSlots - 1) * AHEAD);
#pragma unroll
    for (int i = 0; i < Q_LOADS; ++i) {
        const int r = (int)threadIdx.x / PIECES + i * (kThreads / PIECES);
        const uint4 v = query[i];
        *reinterpret_cast<uint4*>(smem + L::kQueries + r * L::kRow + 16 * (q_piece ^ (r & 7))) =
            make_uint4((v.x & a.q_keep) ^ a.q_flip, (v.y & a.q_keep) ^ a.q_flip, (v.z & a.q_keep) ^ a.q_flip, (v.w & a.q_keep) ^ a.q_flip);
    }
    __syncthreads();

    // lane's row and piece of the matrices that it gives the address of: queries (16 rows, 2 pieces), k (16 rows, 2 pieces, rows first), v
    const int mi = lane >> 3, mr = lane & 7;
    auto at = [&](uint32_t from, int row, int p) { return from + row * L::kRow + 16 * (p ^ (row & 7)); };
    constexpr bool KEEP_Q = D == 64 || (D == 128 && kSlots == 3);      // else they are read again in every step: three CTAs an SM have 168 registers a thread
    uint32_t q[KEEP_Q ? CHUNKS : 1][4];
    if (KEEP_Q) {
#pragma unroll
        for (int d = 0; d < (KEEP_Q ? CHUNKS : 1); ++d) load_matrices(at(queries, mr + 8 * (mi & 1), 2 * d + (mi >> 1)), q[d]);
    }

    auto multiply = [&](uint32_t slot, int step_base, auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        float p[TT][2][4];
#pragma unroll
        for (int i = 0; i < TT; ++i) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) p[i][j][e] = 0.0f;
#pragma unroll
            for (int d = 0; d < CHUNKS; ++d) {
                uint32_t k[4];
                load_matrices(at(slot, 16 * i + mr + 8 * (mi >> 1), 2 * d + (mi & 1)), k);
                if (!KEEP_Q) load_matrices(at(queries, mr + 8 * (mi & 1), 2 * d + (mi >> 1)), q[0]);
                const uint32_t(&x)[4] = q[KEEP_Q ? d : 0];
                mma16<T>(p[i][0], x[0], x[1], x[2], x[3], k[0], k[1]);
                mma16<T>(p[i][1], x[0], x[1], x[2], x[3], k[2], k[3]);
            }
        }
        // ---- softmax.  The running maximum is one of the rounded products that it is subtracted from, so that nothing is above it however large
        // the scores are.
        float alpha[2];
        bool grown = false;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < TT; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& x = p[i][j][2 * r + e];
                        x = __fmul_rn(x, a.scale_log2);
                        const int row = step_base + 16 * i + 8 * j + 2 * c + e;
                        if (MASKED && (row >= limit[r] || row < start)) x = -INFINITY;
                        top = fmaxf(top, x);
                    }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float now = fmaxf(m[r], top), ref = now == -INFINITY ? 0.0f : now;      // a query may have seen nothing yet
            alpha[r] = exp2_fast(m[r] - ref);
            grown = grown || now != m[r];
            m[r] = now;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < TT; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& x = p[i][j][2 * r + e];
                        x = exp2_fast(x - ref);
                        sum += x;
                    }
            l[r] = fmaf(l[r], alpha[r], sum);
        }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int d = 0; d < D / 8; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[d][e] *= alpha[e >> 1];
        }
        // ---- O += P V, P in two parts
#pragma unroll
        for (int i = 0; i < TT; ++i) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {                 // rows 8 * (w / 2) + 2c of queries g + 8 * (w % 2)
                const float x0 = p[i][w >> 1][2 * (w & 1)], x1 = p[i][w >> 1][2 * (w & 1) + 1];
                hi[w] = F16Bits<T>::pack(x0, x1);
                lo[w] = F16Bits<T>::pack(x0 - F16Bits<T>::lo(hi[w]), x1 - F16Bits<T>::hi(hi[w]));
            }
#pragma unroll
            for (int d = 0; d < CHUNKS; ++d) {
                uint32_t v[4];
                load_matrices_transposed(at(slot + L::kV, 16 * i + mr + 8 * (mi & 1), 2 * d + (mi >> 1)), v);
                if (MASKED && fewest < most) {            // this lane's values of rows 2c, 2c + 1 and 8 more
                    constexpr uint32_t E = F16Bits<T>::kInf;
#pragma unroll
                    for (int w = 0; w < 4; ++w)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int row = step_base + 16 * i + 8 * (w & 1) + 2 * c + e;
                            if (row >= fewest && ((v[w] >> (16 * e)) & 0x7fffu) >= E) {
                                atomicOr(noted, 1u << (row - fewest));
                                v[w] &= e ? 0x0000ffffu : 0xffff0000u;
                            }
                        }
                }
                mma16<T>(o[2 * d], hi[0], hi[1], hi[2], hi[3], v[0], v[1]);
                mma16<T>(o[2 * d + 1], hi[0], hi[1], hi[2], hi[3], v[2], v[3]);
                mma16<T>(o[2 * d], lo[0], lo[1], lo[2], lo[3], v[0], v[1]);
                mma16<T>(o[2 * d + 1], lo[0], lo[1], lo[2], lo[3], v[2], v[3]);
            }
        }
    };

    int in = kSlots - 1, out = 0;
    for (; base < last; base += AHEAD) {
        const int ahead = base + (kSlots - 1) * AHEAD;
        if (ahead < last) fill(ring + in * L::kSlot, ahead, next);        // into the slot that every lane left at the end of the step before
        commit_copies();
        next = pages_of(ahead + AHEAD);
        in = in + 1 == kSlots ? 0 : in + 1;
        wait_copies<kSlots - 1>();
        __syncwarp();
        if (base >= start && base + STEP <= unmasked) multiply(ring + out * L::kSlot, base, std::false_type{});
        else multiply(ring + out * L::kSlot, base, std::true_type{});
        __syncwarp();
        out = out + 1 == kSlots ? 0 : out + 1;
    }
    wait_copies<0>();

    // ---- the warps' results into one
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if (c == 0) {
            warp_m[warp * kCols + g + 8 * r] = m[r];
            warp_l[warp * kCols + g + 8 * r] = l[r];
        }
    }
    __syncthreads();                                      // every warp has left its ring, too
    if (threadIdx.x < kCols) {
        const int col = threadIdx.x;
        float top = -INFINITY, total = 0.0f;
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, warp_m[w * kCols + col]);
        for (int w = 0; w < kWarps; ++w)
            if (warp_l[w * kCols + col] != 0.0f) total += warp_l[w * kCols + col] * exp2_fast(warp_m[w * kCols + col] - top);
        cta_m[col] = top;
        cta_l[col] = total;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int col = g + 8 * r;
        const float w = m[r] == -INFINITY ? 0.0f : exp2_fast(m[r] - cta_m[col]);
        float* const dst = buf + (warp * kCols + col) * BUF + 2 * c;
        if (col < qt.rows)
#pragma unroll
            for (int d = 0; d < D / 8; ++d) *reinterpret_cast<float2*>(dst + 8 * d) = make_float2(o[d][2 * r] * w, o[d][2 * r + 1] * w);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < qt.rows * (D / 4); i += kThreads) {
        const int col = i / (D / 4), d = i % (D / 4) * 4;
        float4 x = *reinterpret_cast<const float4*>(buf + col * BUF + d);
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
            const float4 y = *reinterpret_cast<const float4*>(buf + (w * kCols + col) * BUF + d);
            x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
        }
        for (unsigned w = *noted; w; w &= w - 1) {
            const int row = fewest + __ffs(w) - 1;
            if (row >= rows_seen(s, position, token_of(col)) || row < start) continue;
            float* const e = reinterpret_cast<float*>(&x);
            for (int k = 0; k < 4; ++k) e[k] += not_finite<T, true>(a, pages, row, h, d + k);
        }
        *reinterpret_cast<float4*>(sums + col * D + d) = x;
    }
    __syncthreads();

    auto query_at = [&](int col) {                        // token * Hq + head
        const int t = token_of(col);
        return (int64_t)(qt.token0 + t) * a.Hq + h * a.G + (qt.row0 + col - t * a.G);
    };
    if (a.mark && share == 0 && threadIdx.x < (unsigned)qt.rows) a.part.stats[query_at(threadIdx.x)] = make_float2(0.0f, kWritten);
    auto store = [&](int col, int d, float x, float y) {
        *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + query_at(col) * D + d) = F16Bits<T>::pack(x, y);
    };
    if (a.shares == 1) {
        for (int i = threadIdx.x; i < qt.rows * (D / 2); i += kThreads) {
            const int col = i / (D / 2), d = i % (D / 2) * 2;
            const float total = cta_l[col], inv = total == 0.0f ? 0.0f : 1.0f / total;
            store(col, d, sums[col * D + d] * inv, sums[col * D + d + 1] * inv);
        }
        if (a.by_length && blockIdx.x == 0) wait_predecessor();
        return;
    }
    if (a.shares > kClusterShares) {
        for (int i = threadIdx.x; i < qt.rows * (D / 4); i += kThreads) {
            const int col = i / (D / 4), d = i % (D / 4) * 4;
            *reinterpret_cast<float4*>(a.part.sums + (share * a.part.rows + query_at(col)) * D + d) = *reinterpret_cast<const float4*>(sums + col * D + d);
        }
        if (threadIdx.x < (unsigned)qt.rows)
            a.part.stats[share * a.part.rows + query_at(threadIdx.x)] = make_float2(cta_m[threadIdx.x], cta_l[threadIdx.x]);
        return;
    }
    const cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (threadIdx.x < (unsigned)qt.rows) {
        const int col = threadIdx.x;
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
        for (int r = 0; r < kClusterShares; ++r) weight[r * kCols + col] = ms[r] * inv;
    }
    __syncthreads();
    const int pairs = qt.rows * (D / 2), part = (pairs + a.shares - 1) / a.shares;
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
                x = fmaf(v[r].x, weight[r * kCols + col], x);
                y = fmaf(v[r].y, weight[r * kCols + col], y);
            }
        store(col, d, x, y);
    }
    cluster.sync();                                       // the others read this CTA's sums
    if (a.by_length && blockIdx.x == 0) wait_predecessor();
}

// Joins the shares of one query: a CTA of four times D threads, a quarter of the shares each.
template <typename T, int D>
__global__ void __launch_bounds__(4 * D) paged_join_kernel(const Partials p, int shares, T* out) {
    __shared__ float weight[kMaxShares];
    __shared__ float sum[4][D];
    after_predecessor();
    const int64_t row = blockIdx.x;
    const float2* const stats = p.stats + row;
    if (stats[0].y == kWritten) return;
    const int d = threadIdx.x % D, part = threadIdx.x / D;
    if (threadIdx.x < 32) {
        float top = -INFINITY, total = 0.0f;
        float2 s[kMaxShares / 32];
#pragma unroll
        for (int i = 0; i < kMaxShares / 32; ++i) {
            const int k = threadIdx.x + 32 * i;
            s[i] = k < shares ? stats[k * p.rows] : make_float2(-INFINITY, 0.0f);
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
        for (int i = 0; i < kMaxShares / 32; ++i) weight[threadIdx.x + 32 * i] = s[i].y != 0.0f ? s[i].x * inv : -1.0f;
    }
    __syncthreads();
    const int per = (shares + 3) / 4, first = part * per, last = min(shares, first + per);
    const float* const src = p.sums + row * D + d;
    float x = 0.0f;
    for (int k0 = first; k0 < last; k0 += 8) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)                       // a share that saw nothing may have left no sums
            v[k] = k0 + k < last && weight[k0 + k] != -1.0f ? src[(k0 + k) * p.rows * D] : 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k0 + k < last) x = fmaf(v[k], weight[k0 + k], x);
    }
    sum[part][d] = x;
    __syncthreads();
    if (part > 0) return;
    reinterpret_cast<unsigned short*>(out)[row * D + d] = (unsigned short)F16Bits<T>::pack((sum[0][d] + sum[1][d]) + (sum[2][d] + sum[3][d]), 0.0f);
}

// The same for few shares and any number of queries: a warp each, whose lanes know a share's weight and have 2, 4 or 8 features.
constexpr int kFewShares = 16, kJoinWarps = 4;
template <typename T, int D>
__global__ void __launch_bounds__(32 * kJoinWarps) paged_join_few_kernel(const Partials p, int shares, T* out) {
    constexpr int V = D / 32;
    after_predecessor();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * kJoinWarps + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    const float2 mine = lane < shares ? p.stats[lane * p.rows + row] : make_float2(-INFINITY, 0.0f);
    if (__shfl_sync(0xffffffffu, mine.y, 0) == kWritten) return;
    float top = mine.x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float w = mine.y != 0.0f ? exp2_fast(mine.x - top) : 0.0f;
    float total = w * mine.y;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    const float weight = mine.y != 0.0f ? w * (total == 0.0f ? 0.0f : 1.0f / total) : -1.0f;
    float x[V] = {};
    const float* const src = p.sums + row * D + lane * V;
#pragma unroll 4
    for (int k = 0; k < shares; ++k) {
        const float wk = __shfl_sync(0xffffffffu, weight, k);
        if (wk == -1.0f) continue;                        // a share that saw nothing may have left no sums
        float v[V];
        if constexpr (V == 2) {
            const float2 y = *reinterpret_cast<const float2*>(src + k * p.rows * D);
            v[0] = y.x, v[1] = y.y;
        } else {
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                const float4 y = *reinterpret_cast<const float4*>(src + k * p.rows * D + i);
                v[i] = y.x, v[i + 1] = y.y, v[i + 2] = y.z, v[i + 3] = y.w;
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = fmaf(v[i], wk, x[i]);
    }
    uint32_t* const dst = reinterpret_cast<uint32_t*>(out + row * D + lane * V);
#pragma unroll
    for (int i = 0; i < V; i += 2) dst[i / 2] = F16Bits<T>::pack(x[i], x[i + 1]);
}

struct Plan {
    bool many;
    bool both;                   // sequences of few and of many queries in one batch: a kernel for each
    int rows;                    // queries of a tile
    int64_t tiles, shares, few_shares;
};
// How many shares the rows are divided into, for the kernel of few queries.  Time is counted in rows of a CTA among as many as the SMs hold (36 ns at
// D 128): a round of CTAs takes a share's rows and kSetUp more (latency until the first rows are there, and the join), a last round that is not full its part, but
// no less than kAlone, because few CTAs cannot draw all of the memory's bandwidth.  (D 128, us: 16 sequences of 8192 rows on 8 heads in 1, 2, 3, 4, 5, 6
// shares: 124, 107, 111, 133, 117, 111; 32 of 4096: 104, 134, 105, 117, 122, 118; 100 of 1000: 87, 94, 103.)  Long tables, whose sequences may
// differ much in length, have shares of 2048 rows at most (32 sequences of 1 to 8192 rows: 174, 109, 107, 101, 100, 101), more than a cluster's eight a
// second kernel.  Those are few sequences, one round of CTAs at most: two an SM, which come out even (131072 rows, 8 heads: 296 CTAs 88 to 90 us, 440 of
// three an SM 93 to 104).
// The table's room is all that the host knows of the lengths.  Sequences much shorter than that have shares of a few rows each (32 sequences of 600 rows on 8
// heads: 20 us with tables of 600 rows, 22 of 4096, 43 of 32768 and more; 8 of 2000: 18, 29 of 131072).
int64_t few_shares(int64_t ctas, int64_t D, int64_t max_len, int64_t most) {
    const int64_t step = kWarps * 16 * (D == 64 ? kSubSteps<64> : D == 128 ? kSubSteps<128> : kSubSteps<256>);
    const int64_t sms = sm_count(), set_up = 12800 / D;
    const int64_t useful = (max_len + step - 1) / step, least = max_len / 2048;
    int64_t best = 1, best_cost = 0;
    for (int64_t s = least < 1 ? 1 : least > kClusterShares ? kClusterShares : least; s <= most && (s <= useful || s == 1); ++s) {
        const int64_t slots = sms * (D == 256 ? 1 : s > kClusterShares ? kSingleRound : kResident<128>), alone = (D == 256 ? 80 : 45) * slots / 100;
        const int64_t n = ctas * s, left = n % slots;
        const int64_t rounds = n / slots * slots + (left == 0 ? 0 : s > kClusterShares ? slots : left < alone ? alone : left);
        const int64_t cost = rounds * (max_len / s + set_up) + (s > kClusterShares ? slots * set_up : 0);
        if (best_cost == 0 || cost < best_cost) best = s, best_cost = cost;
        if (n > 16 * slots) break;
    }
    return best < most ? best : most;
}
Plan plan_of(int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_len, bool packed) {
    // One tile of few queries reads the cache as fast as it comes; a second one reads it again, and a CTA of the other kernel is no slower for up to 256.  (32
    // sequences of 4096 rows, 8 heads, few and many: 16 queries of each 112 and 127 us, 20: 160 and 127, 32: 156 and 127.)
    const int64_t G = Hq / Hkv;
    Plan p{};
    p.many = packed ? N > B && N * G > kCols * B : N / B * G > kCols;
    // The host cannot tell tokens that belong to nobody from parts of prompts: they bring the other kernel's launch along (32 sequences of 600 rows 20 us, 28 with
    // 7 such tokens) and bound the shares of few queries to a cluster's (one sequence of 131072 rows 90 us, 254 to 311).
    p.both = packed && N > B && G <= kCols;
    p.many = p.many || p.both;
    p.rows = p.many ? paged_many_tile(D) : kCols;
    p.tiles = tile_count(B, N, G, p.rows, packed);
    p.few_shares = few_shares(p.both ? (B + 1) * Hkv : p.tiles * Hkv, D, max_len, p.both ? kClusterShares : kMaxShares);
    p.shares = p.few_shares;
    if (p.many) {
        // A CTA an SM.  Shares beyond one round of CTAs do not pay for what they write and for the join, even where the rounds do not come out even.  (2048
        // tokens of 32 heads, D 128: 256 CTAs of 32768 rows 891 us in 1 share, 936 in 2, 946 in 4; 256 of 8192 rows 227, 270, 287.)  Within a round a share takes 14 ns a row, and more than one 3 us for the join and what they write and it reads at 6 bytes a
        // ns.  (64 tokens behind 2000 rows, 32 heads on 8: 36 us in 1 share, 16 in 7; 512 tokens from the first on: 15 in 1, 20 in 2.)  What may be
        // tiles of few queries is not counted where those have a kernel of their own.
        const int64_t ctas = (p.both ? N * G / p.rows + 1 : p.tiles) * Hkv;
        int64_t most = sm_count() / ctas, best = 0;
        if (most > max_len / kShareRows) most = max_len / kShareRows;
        if (most > kMaxShares) most = kMaxShares;
        p.shares = 1;
        for (int64_t s = 1; s <= most; ++s) {
            const int64_t ns = 14 * max_len / s + (s > 1 ? 3000 + s * (N * Hq) * D * 8 / 6000 : 0);
            if (s == 1 || ns < best) best = ns, p.shares = s;
        }
    }
    return p;
}
bool through_workspace(const Plan& p) { return p.many ? p.shares > 1 : p.shares > kClusterShares; }

template <typename T, int D, int SLOTS>
int launch_slots(const PagedAttnArgs& a, cudaStream_t st) {
    constexpr int smem = Smem<D, SLOTS>::kBytes;
    static SmemOptIn opt_in;
    if (int rc = opt_in.ensure(paged_few_kernel<T, D, SLOTS>, smem)) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((int64_t)a.tiles * a.Hkv * a.shares));
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
    BI8_CUDA_TRY(cudaLaunchKernelEx(&cfg, paged_few_kernel<T, D, SLOTS>, a));
    return BI8_OK;
}
template <typename T, int D>
int launch(const PagedAttnArgs& a, cudaStream_t st) {
    if constexpr (D != 256)
        if (a.shares > kClusterShares) return launch_slots<T, D, 3>(a, st);
    return launch_slots<T, D, 2>(a, st);
}

template <typename T>
int join(const Partials& p, int shares, void* out, int64_t D, cudaStream_t st) {
    T* const o = static_cast<T*>(out);
    if (shares <= kFewShares) {
        const unsigned grid = (unsigned)((p.rows + kJoinWarps - 1) / kJoinWarps);
        if (D == 64) return launch_chained(paged_join_few_kernel<T, 64>, grid, 32 * kJoinWarps, 0, st, p, shares, o);
        if (D == 128) return launch_chained(paged_join_few_kernel<T, 128>, grid, 32 * kJoinWarps, 0, st, p, shares, o);
        return launch_chained(paged_join_few_kernel<T, 256>, grid, 32 * kJoinWarps, 0, st, p, shares, o);
    }
    if (D == 64) return launch_chained(paged_join_kernel<T, 64>, (unsigned)p.rows, 256, 0, st, p, shares, o);
    if (D == 128) return launch_chained(paged_join_kernel<T, 128>, (unsigned)p.rows, 512, 0, st, p, shares, o);
    return launch_chained(paged_join_kernel<T, 256>, (unsigned)p.rows, 1024, 0, st, p, shares, o);
}

}  // namespace

int launch_paged_join(const Partials& p, int shares, void* out, int dt, int64_t D, cudaStream_t st) {
    return dt == BI8_BF16 ? join<__nv_bfloat16>(p, shares, out, D, st) : join<__half>(p, shares, out, D, st);
}

int launch_paged_few(const PagedAttnArgs& a, int dt, int64_t D, cudaStream_t st) {
    auto go = [&](auto* tag) {
        using E = std::remove_pointer_t<decltype(tag)>;
        if (D == 64) return launch<E, 64>(a, st);
        if (D == 128) return launch<E, 128>(a, st);
        return launch<E, 256>(a, st);
    };
    return dt == BI8_BF16 ? go(static_cast<__nv_bfloat16*>(nullptr)) : go(static_cast<__half*>(nullptr));
}

size_t attention_paged_workspace_bytes(int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_len, bool packed) {
    const Plan p = plan_of(B, N, Hq, Hkv, D, max_len, packed);
    return through_workspace(p) ? (size_t)(p.shares * N * Hq) * (D + 2) * 4 : 0;
}

int launch_attention_paged(const void* q, int dt, int64_t q_tok, int64_t q_head, const bi8_paged_cache* cache, const Sequences& seq, float scale, void* out,
                           int64_t Hq, int64_t D, void* workspace, cudaStream_t st) {
    const int64_t Hkv = cache->heads, G = Hq / Hkv;
    const Plan p = plan_of(seq.B, seq.N, Hq, Hkv, D, seq.max_len, seq.cu != nullptr);
    if (p.tiles * Hkv * p.shares > 0x7fffffff || ((int64_t)seq.B + 1) * Hkv * p.few_shares > 0x7fffffff || (int64_t)seq.N * Hq > 0x7fffffff)
        return fail(BI8_ERR_LIMIT, "attention_paged: %lld queries exceed one launch", (long long)seq.N * Hq);
    if (cache->pages == 0) {                                  // whatever a query sees reads as zeros
        BI8_CUDA_TRY(cudaMemsetAsync(out, 0, (size_t)seq.N * Hq * D * 2, st));
        return BI8_OK;
    }
    PagedAttnArgs a{};
    a.q = q;
    a.q_tok = q_tok;
    a.q_head = q_head;
    a.cache = *cache;
    a.seq = seq;
    a.out = out;
    a.part.rows = (int64_t)seq.N * Hq;
    a.part.sums = static_cast<float*>(workspace);
    a.part.stats = reinterpret_cast<float2*>(a.part.sums + p.shares * a.part.rows * D);
    a.Hq = (int)Hq;
    a.Hkv = (int)Hkv;
    a.G = (int)G;
    a.scale_log2 = std::fmax(std::fabs(scale) * 1.4426950408889634f, 0x1p-149f);       // never 0, which the infinities of unseen rows do not bear
    a.q_keep = scale == 0.0f ? 0u : 0xffffffffu;
    a.q_flip = scale < 0.0f ? 0x80008000u : 0u;
    a.group = FastDiv(G);
    a.heads = FastDiv(Hkv);
    a.sequences = FastDiv(seq.B);
    a.by_length = p.both;
    const bool joined = through_workspace(p);
    if (p.many) {
        a.shares = (int)p.shares;
        a.tiles = (int)p.tiles;
        a.per_share = FastDiv(p.shares);
        a.per_sequence = FastDiv(seq.cu ? 1 : ((int64_t)seq.T * G + p.rows - 1) / p.rows);
        if (int rc = launch_paged_many(a, dt, D, st)) return rc;
    }
    if (!p.many || p.both) {
        PagedAttnArgs f = a;
        f.shares = (int)p.few_shares;
        f.tiles = (int)(p.both ? seq.B + 1 : p.tiles);
        f.mark = p.both && joined;
        f.per_share = FastDiv(p.few_shares);
        f.per_sequence = FastDiv(seq.cu ? 1 : ((int64_t)seq.T * G + kCols - 1) / kCols);
        if (int rc = launch_paged_few(f, dt, D, st)) return rc;
    }
    return joined ? launch_paged_join(a.part, (int)p.shares, out, dt, D, st) : BI8_OK;
}

}  // namespace bi8
