// Attention of many queries of each cache head over a paged 16-bit cache: parts of prompts, alone or among single tokens.  The same mathematics as
// in paged_attention.cu, on tcgen05.
//
// A CTA takes up to two tiles of 128 queries (tokens and the G heads that share a cache head, in that order) of one sequence and streams the sequence's
// rows past them, kRows at a time.  One warp fetches k and v by TMA (boxes of as many rows as surely lie in one page, 128-byte swizzle), one
// issues the products, two look after what v holds where it must not count, and four warps a tile, one thread a query, do the softmax:
//   S = Q K^T    queries and keys from shared memory, scores in tensor memory
//   P = 2^(c S - m)  by the query's thread, back into the scores' own tensor memory as 16-bit numbers
//   O += P V     weights from tensor memory, values from shared memory as they lie (the contraction runs over their rows)
// While one tile's weights are computed the other's products run.  With heads of 256 features there is room for one tile, whose scores have two
// places instead.
//
// The maximum m that a query subtracts follows its scores only when they have grown by 2^8 (fp32 sums and 16-bit weights lose nothing by
// being that much larger), so that O is hardly ever rescaled; that is done by the query's own thread.  m is a rounded number, subtracted inside one
// multiply-add: all weights are relative to the same power of two, whatever it is.  Only where scores are so large (2^20) that its rounding is
// a power of two of its own the differences of scores are taken first; the scores' own rounding is no smaller then.
//
// What bounds it: the chain of a tile, scores read (545 cycles a step with their maximum), weights (1460 alone, 1900 beside the other tile's: the exponentials'
// unit has 1024 for each), the rest of the product and the next scores (1080), 3540 cycles in all of which the tensor cores work 2048 (without any
// exponentials a call takes 7 % less); the power cap; and whole rounds of CTAs.  2048 tokens, the last of 32768 rows, 32 heads on 8 of 128 features, are 256 CTAs for
// 148 SMs: 880 us alone, 990 to 1010 in a loop (1.06 PFLOP/s, 75 % of cuBLAS's sustained rate).  With heads of 64 a step is no shorter, although its products are half: 8 x 512
// tokens over 2048 rows, 32 heads, 131 us, the exponentials' unit busy half of the time, the tensor cores a quarter.  Heads of 256, one tile a CTA: 2048 tokens, the
// last of 16384 rows, 32 heads on 8, 1090 to 1170 us for 620 of products.  Tried without gain: a part of the exponentials as polynomials on the multiply-add pipe, two threads a query, steps of 64 rows
// with two places for the scores of heads of 64.
//
// Weights are 16-bit numbers: a rounding of half a step each, at random, which leaves the result about as much error again as its own rounding (against 64
// bits 0.0023 in the 2-norm for bf16, 0.0017 by its rounding alone).  A second product with what they lose would cost half of the time again.  Their total is
// summed before they are rounded, in fp32.
//
// What a query does not see must not count: scores are masked, and v's rows before the start and behind the last one are overwritten by zeros in
// shared memory before the product, since 0 times an infinity is none.  Infinities and NaN of rows that only some queries see take a way of
// their own (paged_attention.cuh).
#include "paged_attention.cuh"
#include "tc_common.cuh"

#include <atomic>
#include <type_traits>

namespace bi8 {
namespace {

using namespace ptx;

constexpr int kTileRows = 128;
constexpr int kSoftmaxRegisters = 208, kOtherRegisters = 80;       // of two tiles' warps and of the four others

template <int D>
struct Shape {
    static constexpr int kTiles = D == 256 ? 1 : 2;                  // of queries
    static constexpr int kRows = D == 256 ? 64 : 128;                // of the cache at a time
    static constexpr int kStages = D == 64 ? 8 : 5;
    static constexpr int kAhead = kTiles == 1 ? 2 : 1;               // scores that are under way before the first weights are used
    static constexpr int kWarps = 4 * kTiles + 4, kThreads = 32 * kWarps;
    static constexpr int kQTile = kTileRows * D * 2, kStage = kRows * D * 2;
    static constexpr int kScores = 0, kOut = 2 * kRows;              // columns of tensor memory
    static constexpr int kColumns = 512;
    static_assert(kOut + kTiles * D <= kColumns, "tensor memory");
    // barriers
    static constexpr int kFull = 0, kEmpty = kStages, kScoresFull = 2 * kStages, kWeightsFull = kScoresFull + 2, kProductDone = kWeightsFull + 4,
                         kQueries = kProductDone + 2, kClean = kQueries + 2, kEnd = kClean + kStages, kBarriers = kEnd + 1;
    static constexpr int kStagesAt = kTiles * kQTile, kBarriersAt = kStagesAt + kStages * kStage, kMisc = kBarriersAt + 8 * kBarriers;
    static constexpr int kNoted = kMisc + 16, kBytes = kNoted + 32 + 1024;     // tensor memory's address, abort flag, a word that stays zero; rows noted; alignment
};

template <typename T, int D>
__global__ void __launch_bounds__(Shape<D>::kThreads, 1)
    paged_many_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const PagedAttnArgs a, const int box_rows, const int share_rows,
                      int* status, const long long wait_limit) {
    using Z = Shape<D>;
    constexpr int KT = Z::kRows, TILES = Z::kTiles, CHUNKS = D / 64;
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int MMA_WARP = 4 * TILES, LOAD_WARP = MMA_WARP + 1;
    auto bar = [&](int i) { return base + (uint32_t)(Z::kBarriersAt + 8 * i); };
    const uint32_t holder = base + Z::kMisc, abort_flag = holder + 4, zero_word = holder + 8;

    const int tile_head = (int)a.per_share.div(blockIdx.x), share = (int)blockIdx.x - tile_head * a.shares;
    const int turn = (int)a.heads.div((unsigned)tile_head), h = tile_head - turn * a.Hkv;
    if (warp == LOAD_WARP && lane == 0) {
        prefetch_map(&k_map);
        prefetch_map(&v_map);
    }
    after_predecessor();
    const Sequences& s = a.seq;
    // A sequence's last tiles see the most rows: they go first, so that short ones fill what is left at the end.
    int tile_index = a.tiles - 1 - turn;
    if (!s.cu) {
        const int before = (int)a.sequences.div((unsigned)turn);
        tile_index = (turn - before * s.B) * (int)a.per_sequence.d + ((int)a.per_sequence.d - 1 - before);
    }
    const QueryTile qt = find_tile(s, tile_index, a.G, TILES * kTileRows, a.per_sequence);
    if (qt.rows == 0 || (a.by_length && (int64_t)qt.n * a.G <= kFewQueries)) return;
    auto token_of = [&](int r) { return (int)a.group.div((unsigned)(qt.row0 + r)); };
    auto query_at = [&](int r) {                              // token * Hq + head
        const int t = token_of(r);
        return (int64_t)(qt.token0 + t) * a.Hq + h * a.G + (qt.row0 + r - t * a.G);
    };

    // ---- the tiles' queries are on their way while the rest is found out: neighbouring threads have neighbouring pieces
    constexpr int PIECES = D / 8, Q_ROWS = 128 / PIECES, Q_LOADS = PIECES < 16 ? PIECES : 16;
    const int tiles = qt.rows > kTileRows ? 2 : 1, my_tile = warp / 4, q_row = (threadIdx.x & 127) / PIECES, q_piece = threadIdx.x % PIECES;
    auto load_query = [&](int row) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        const int r = my_tile * kTileRows + row;
        if (r < qt.rows) {
            const int tok = token_of(r), head = h * a.G + (qt.row0 + r - tok * a.G);
            v = ld_nc_v4(static_cast<const T*>(a.q) + (int64_t)(qt.token0 + tok) * a.q_tok + head * a.q_head + 8 * q_piece);
        }
        return v;
    };
    uint4 query[Q_LOADS];
    if (my_tile < tiles && warp < MMA_WARP) {
#pragma unroll
        for (int i = 0; i < Q_LOADS; ++i) query[i] = load_query(q_row + i * Q_ROWS);
    }

    // ---- rows of this share.  A tile takes as many shares as its rows fill.
    const long long position = s.first_position(qt.b, qt.n);
    const int fewest = rows_seen(s, position, token_of(0)), most = rows_seen(s, position, token_of(qt.rows - 1));
    const int start = s.start(qt.b), origin = start & -box_rows, n_rows = most > start ? most - origin : 0;
    const int count = max(1, min(a.shares, n_rows / share_rows));
    const int chunk = (n_rows + count * KT - 1) / (count * KT) * KT;
    const int first = origin + min(n_rows, share * chunk), last = share < count ? min(origin + n_rows, first + chunk) : first;
    const int steps = (last - first + KT - 1) / KT;
    if (steps == 0) {                                         // nothing to see, or no such share
        for (int r = threadIdx.x; r < qt.rows; r += Z::kThreads) {
            if (a.shares > 1) a.part.stats[share * a.part.rows + query_at(r)] = make_float2(-INFINITY, count == 1 && share == 0 ? kWritten : 0.0f);
            if (count == 1 && share == 0) {
                uint4* const dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + query_at(r) * D);
                for (int i = 0; i < D / 8; ++i) dst[i] = make_uint4(0u, 0u, 0u, 0u);
            }
        }
        return;
    }

    // the pages of the first step's rows, a lane of the loading warp for every box
    const int* const table = s.pages + (qt.b < s.B ? qt.b : 0) * s.pages_step;
    int first_page = 0;
    if (warp == LOAD_WARP && lane < KT / box_rows && first + lane * box_rows < last) first_page = table[s.page.div((unsigned)(first + lane * box_rows))];

    // ---- set-up
    if (warp == MMA_WARP) {
        tmem_alloc(holder, Z::kColumns);
        tmem_relinquish();
        if (lane == 0) {
            sts_u32(abort_flag, 0u);
            sts_u32(zero_word, 0u);
            for (int i = 0; i < Z::kStages; ++i) {
                mbar_init(bar(Z::kFull + i), 1);
                mbar_init(bar(Z::kEmpty + i), 1);
                mbar_init(bar(Z::kClean + i), 2);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(bar(Z::kScoresFull + i), 1);
                mbar_init(bar(Z::kWeightsFull + i), 128);
                mbar_init(bar(Z::kWeightsFull + 2 + i), 128);
                mbar_init(bar(Z::kProductDone + i), 1);
                mbar_init(bar(Z::kQueries + i), 128);
            }
            mbar_init(bar(Z::kEnd), 1);
            mbar_fence_init();
        }
        if (lane < 8) sts_u32(base + Z::kNoted + 4 * lane, 0u);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = lds_u32(holder);
    auto stage_at = [&](int stage) { return base + (uint32_t)(Z::kStagesAt + stage * Z::kStage); };
    // where k and v of a step come in the order of the copies
    auto order_v = [&](int j) { return min(steps, j + Z::kAhead) + j; };
    auto order_k = [&](int j) { return j < Z::kAhead ? j : order_v(j - Z::kAhead) + 1; };

    if (warp >= MMA_WARP) {
        if constexpr (TILES == 2) setmaxnreg_dec<kOtherRegisters>();
        if (warp == LOAD_WARP) {
            // ---- copies: a box of box_rows rows and 64 features at a time, a lane for every box_rows rows of the step
            const int boxes = KT / box_rows;
            bool ok = true;
            int order = 0;
            auto fetch = [&](const CUtensorMap& map, int j) {
                const int stage = order % Z::kStages, parity = (order / Z::kStages) & 1;
                const int row = first + j * KT + lane * box_rows;
                const bool mine = lane < boxes && row < last;
                const int in_table = mine ? (int)s.page.div((unsigned)row) : 0;
                const int page = j == 0 ? first_page : mine ? table[in_table] : 0;
                ok = __all_sync(0xffffffffu, mbar_wait(bar(Z::kEmpty + stage), (uint32_t)parity ^ 1u, abort_flag, wait_limit));
                if (!ok) {
                    if (lane == 0) report_timeout(status, abort_flag, W_EMPTY_AB);
                    return;
                }
                const int copied = __popc(__ballot_sync(0xffffffffu, mine));
                if (lane == 0) mbar_expect_tx(bar(Z::kFull + stage), (uint32_t)(copied * box_rows * D * 2));
                __syncwarp();
                if (mine) {
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c)
                        tma_load_4d(stage_at(stage) + (uint32_t)((c * KT + lane * box_rows) * 128), &map, bar(Z::kFull + stage), 64 * c, row - in_table * (int)s.page.d, h, page);
                }
                __syncwarp();
                ++order;
            };
            for (int j = 0; j < min(Z::kAhead, steps) && ok; ++j) fetch(k_map, j);
            for (int j = 0; j < steps && ok; ++j) {
                fetch(v_map, j);
                if (ok && j + Z::kAhead < steps) fetch(k_map, j + Z::kAhead);
            }
            // after an abort: the copies that are still on their way
            if (!ok)
                for (int i = max(0, order - Z::kStages); i < order; ++i) (void)mbar_wait(bar(Z::kFull + i % Z::kStages), (uint32_t)(i / Z::kStages) & 1u, zero_word, wait_limit);
        } else if (warp == MMA_WARP) {
            // ---- products, issued by one thread
            if (elect_one()) {
                constexpr uint32_t S_DESC = umma_idesc_16bit(kTileRows, KT, BF16, false), O_DESC = umma_idesc_16bit(kTileRows, D, BF16, true);
                bool ok = true;
                auto wait = [&](int b, int parity, int code) {
                    if (!ok) return;
                    ok = mbar_wait(bar(b), (uint32_t)parity, abort_flag, wait_limit);
                    if (!ok) report_timeout(status, abort_flag, code);
                };
                auto wait_stage = [&](int order) { wait(Z::kFull + order % Z::kStages, (order / Z::kStages) & 1, W_FULL_AB); };
                auto scores = [&](int t, int buf, int order) {
                    const uint32_t q = base + (uint32_t)(t * Z::kQTile), k = stage_at(order % Z::kStages);
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)
                        mma_f16(tmem + (uint32_t)(Z::kScores + buf * KT), umma_desc_k_sw128(q + (uint32_t)((i / 4) * kTileRows * 128 + (i % 4) * 32)),
                                umma_desc_k_sw128(k + (uint32_t)((i / 4) * KT * 128 + (i % 4) * 32)), S_DESC, i > 0);
                    tc_commit(bar(Z::kScoresFull + buf));
                };
                for (int t = 0; t < tiles; ++t) wait(Z::kQueries + t, 0, W_FULL_AB);
                for (int j = 0; j < min(Z::kAhead, steps) && ok; ++j) {
                    wait_stage(order_k(j));
                    if (!ok) break;
                    tc_fence_after();
                    for (int t = 0; t < tiles; ++t) scores(t, TILES == 2 ? t : j & 1, order_k(j));
                    tc_commit(bar(Z::kEmpty + order_k(j) % Z::kStages));
                }
                for (int j = 0; j < steps && ok; ++j) {
                    const int ov = order_v(j), ahead = j + Z::kAhead, ok_order = order_k(ahead);
                    wait_stage(ov);
                    // in every step, so that the warps that look after v are never behind
                    wait(Z::kClean + j % Z::kStages, (j / Z::kStages) & 1, W_FULL_AB);
                    for (int t = 0; t < tiles && ok; ++t) {
                        const int buf = TILES == 2 ? t : j & 1;
                        const uint32_t v = stage_at(ov % Z::kStages);
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            wait(Z::kWeightsFull + 2 * half + buf, TILES == 2 ? j & 1 : (j >> 1) & 1, W_ACC_FULL);
                            if (!ok) break;
                            tc_fence_after();
#pragma unroll
                            for (int i = half * (KT / 32); i < (half + 1) * (KT / 32); ++i)
                                mma_f16_ta(tmem + (uint32_t)(Z::kOut + t * D), tmem + (uint32_t)(Z::kScores + buf * KT + 8 * i), umma_desc_mn_sw128(v + (uint32_t)(2048 * i), KT * 128),
                                           O_DESC, j > 0 || i > 0);
                        }
                        if (!ok) break;
                        tc_commit(bar(Z::kProductDone + t));
                        if (ahead < steps) {
                            if (t == 0) wait_stage(ok_order);
                            if (ok) scores(t, buf, ok_order);
                        }
                    }
                    if (!ok) break;
                    // not behind the last product, whose own barrier is the last that anyone waits for: nothing arrives in memory that the CTA has left
                    if (j + 1 < steps) tc_commit(bar(Z::kEmpty + ov % Z::kStages));
                    if (ahead < steps) tc_commit(bar(Z::kEmpty + ok_order % Z::kStages));
                }
                if (!ok) {                                        // products that are still under way
                    tc_commit(bar(Z::kEnd));
                    (void)mbar_wait(bar(Z::kEnd), 0u, zero_word, wait_limit);
                }
            }
            __syncwarp();
        } else {
            // ---- v's rows that nobody sees become zeros, and those that only some of the queries see are looked through
            const int me = threadIdx.x - 32 * (LOAD_WARP + 1), row0 = me >> 3;
            bool ok = true;
            for (int j = 0; j < steps && ok; ++j) {
                const int order = order_v(j), stage = order % Z::kStages, at = first + j * KT;
                // First the step's scores: they show that whatever the stage held before has come and gone (a wait for a barrier's phase is none while an
                // older one is under way, and copies may overtake one another).
                const int buf = TILES == 2 ? 0 : j & 1;
                ok = __all_sync(0xffffffffu, mbar_wait(bar(Z::kScoresFull + buf), (uint32_t)(TILES == 2 ? j & 1 : (j >> 1) & 1), abort_flag, wait_limit) &&
                                                 mbar_wait(bar(Z::kFull + stage), (uint32_t)(order / Z::kStages) & 1u, abort_flag, wait_limit));
                if (!ok) {
                    if (lane == 0) report_timeout(status, abort_flag, W_FULL_AB);
                    break;
                }
                if (at < start || at + KT > min(last, fewest)) {
                    uint8_t* const v = smem + Z::kStagesAt + stage * Z::kStage;
                    constexpr int LOOKS = 8 * KT / 64;
                    uint32_t largest = 0u;
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll 8
                        for (int i = 0; i < LOOKS; ++i) {
                            uint4* const piece = reinterpret_cast<uint4*>(v + c * KT * 128 + (me + 64 * i) * 16);
                            const int row = at + row0 + 8 * i;
                            if (row < start || row >= last) *piece = make_uint4(0u, 0u, 0u, 0u);
                            else if (row >= fewest) largest = max(largest, absmax8(*piece));
                        }
                    if (__any_sync(0xffffffffu, largest >= F16Bits<T>::kInf)) {
                        for (int i = me; i < CHUNKS * 8 * KT; i += 64) {
                            uint4* const piece = reinterpret_cast<uint4*>(v + i * 16);
                            const int row = at + (i >> 3) % KT;
                            if (row < fewest || absmax8(*piece) < F16Bits<T>::kInf) continue;
                            atomicOr(reinterpret_cast<unsigned*>(smem + Z::kNoted) + ((row - fewest) >> 5), 1u << ((row - fewest) & 31));
                            unsigned short* const value = reinterpret_cast<unsigned short*>(piece);
                            for (int e = 0; e < 8; ++e)
                                if ((value[e] & 0x7fffu) >= F16Bits<T>::kInf) value[e] = 0;
                        }
                    }
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(Z::kClean + j % Z::kStages));      // v may be in any place, so these go by steps
            }
        }
    } else {
        if constexpr (TILES == 2) setmaxnreg_inc<kSoftmaxRegisters>();
        if (warp / 4 < tiles) {
            // ---- softmax: a thread is a query
            const int t = warp / 4, r = t * kTileRows + (threadIdx.x & 127);
            const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21), out = lanes + (uint32_t)(Z::kOut + t * D);
            {
                auto store_query = [&](int row, const uint4& v) {
                    *reinterpret_cast<uint4*>(smem + t * Z::kQTile + (q_piece / 8) * kTileRows * 128 + row * 128 + (((q_piece % 8) ^ (row & 7)) << 4)) =
                        make_uint4((v.x & a.q_keep) ^ a.q_flip, (v.y & a.q_keep) ^ a.q_flip, (v.z & a.q_keep) ^ a.q_flip, (v.w & a.q_keep) ^ a.q_flip);
                };
#pragma unroll
                for (int i = 0; i < Q_LOADS; ++i) store_query(q_row + i * Q_ROWS, query[i]);
                if constexpr (PIECES > Q_LOADS) {
#pragma unroll
                    for (int i = 0; i < Q_LOADS; ++i) query[i] = load_query(q_row + (Q_LOADS + i) * Q_ROWS);
#pragma unroll
                    for (int i = 0; i < Q_LOADS; ++i) store_query(q_row + (Q_LOADS + i) * Q_ROWS, query[i]);
                }
                fence_proxy_async_smem();
                mbar_arrive(bar(Z::kQueries + t));
            }
            const bool live = r < qt.rows;
            const int limit = live ? min(last, rows_seen(s, position, token_of(r))) : last, unmasked = min(last, fewest);
            const float c = a.scale_log2;
            constexpr float kGrowth = 8.0f, kLift = BF16 ? 0.0f : 6.0f;      // fp16 weights: 2^-20 of the largest is still a normal number
            float m = -INFINITY, shift = -INFINITY;                // the score that weights are relative to; c m - kLift as it is subtracted
            float total = 0.0f;
            bool ok = true;
            for (int j = 0; j < steps; ++j) {
                const int buf = TILES == 2 ? t : j & 1, at = first + j * KT;
                const uint32_t scores = lanes + (uint32_t)(Z::kScores + buf * KT);
                const bool masked = at < start || at + KT > unmasked;
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar(Z::kScoresFull + buf), TILES == 2 ? j & 1 : (j >> 1) & 1, abort_flag, wait_limit));
                if (!ok) {
                    if (lane == 0) report_timeout(status, abort_flag, W_ACC_FULL);
                    break;
                }
                tc_fence_after();
                uint32_t x[KT];
#pragma unroll
                for (int i = 0; i < KT; i += 32) tmem_ld32(scores + (uint32_t)i, *reinterpret_cast<uint32_t(*)[32]>(x + i));
                tmem_wait_ld();
                if (masked) {
#pragma unroll
                    for (int i = 0; i < KT; ++i)
                        if (at + i >= limit || at + i < start) x[i] = 0xff800000u;
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < KT; ++i) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(x[i]));
                const float now = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
                const bool need = (now - m) * c > kGrowth;         // a first score always is
                // O is at rest when the product before is done.  With two tiles these scores came after it; with one it is waited for in every step, which also
                // keeps the barrier's phases in sight: a wait for one phase may be one behind, not two.
                if (TILES == 1 && j > 0) {
                    ok = __all_sync(0xffffffffu, mbar_wait(bar(Z::kProductDone), (uint32_t)(j - 1) & 1u, abort_flag, wait_limit));
                    if (!ok) {
                        if (lane == 0) report_timeout(status, abort_flag, W_ACC_EMPTY);
                        break;
                    }
                    tc_fence_after();
                }
                if (__any_sync(0xffffffffu, need)) {
                    float alpha = 1.0f;
                    if (need) {
                        m = now;
                        const float next = __fmaf_rn(m, c, -kLift);
                        alpha = exp2_fast(shift - next);
                        shift = next;
                        total *= alpha;
                    }
                    if (j > 0) {
                        const uint64_t both = pack_f32x2(alpha, alpha);
#pragma unroll
                        for (int d = 0; d < D; d += 16) {
                            uint32_t o[16];
                            tmem_ld16(out + (uint32_t)d, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; i += 2) {
                                float y, z;
                                unpack_f32x2(mul_f32x2(pack_u32x2(o[i], o[i + 1]), both), y, z);
                                o[i] = __float_as_uint(y), o[i + 1] = __float_as_uint(z);
                            }
                            tmem_st16(out + (uint32_t)d, o);
                        }
                    }
                }
                const float zero = m == -INFINITY ? 0.0f : m, ref = m == -INFINITY ? 0.0f : shift;
                const uint64_t cc = pack_f32x2(c, c), less = pack_f32x2(-ref, -ref);
                uint64_t sums[2] = {0ull, 0ull};
                auto weights = [&](auto far) {
#pragma unroll
                    for (int i0 = 0; i0 < KT; i0 += KT / 4) {
                        uint32_t p[KT / 8];
#pragma unroll
                        for (int i = 0; i < KT / 4; i += 2) {
                            float y, z;
                            if (decltype(far)::value) {
                                y = __fmaf_rn(__uint_as_float(x[i0 + i]) - zero, c, -kLift);
                                z = __fmaf_rn(__uint_as_float(x[i0 + i + 1]) - zero, c, -kLift);
                            } else {
                                unpack_f32x2(fma_f32x2(pack_u32x2(x[i0 + i], x[i0 + i + 1]), cc, less), y, z);
                            }
                            y = exp2_fast(y);
                            z = exp2_fast(z);
                            sums[(i >> 1) & 1] = add_f32x2(sums[(i >> 1) & 1], pack_f32x2(y, z));
                            p[i / 2] = F16Bits<T>::pack(y, z);
                        }
                        if (i0 == KT / 2) {
                            tmem_wait_st();
                            tc_fence_before();
                            mbar_arrive(bar(Z::kWeightsFull + buf));
                        }
                        if constexpr (KT == 128) tmem_st16(scores + (uint32_t)(i0 / 2), p);
                        else tmem_st8(scores + (uint32_t)(i0 / 2), p);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    mbar_arrive(bar(Z::kWeightsFull + 2 + buf));
                };
                if (__any_sync(0xffffffffu, fabsf(ref) >= 0x1p20f)) weights(std::true_type{});
                else weights(std::false_type{});
                float y, z;
                unpack_f32x2(add_f32x2(sums[0], sums[1]), y, z);
                total += y + z;
            }
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar(Z::kProductDone + t), (uint32_t)(steps - 1) & 1u, abort_flag, wait_limit));
            if (!ok && lane == 0) report_timeout(status, abort_flag, W_ACC_FULL);
            // The barriers between the parts of the results have no limit of their own.  So a tile's four warps, all of which get here because every wait before
            // this one ends, go on to them together or not at all: one may have run out of time, or seen that others did, where the next had what it waited for.
            if (role_barrier_all(t + 1, 128, ok)) {
                // ---- results
                tc_fence_after();
                const bool whole = count == 1;
                const float inv = total == 0.0f ? 0.0f : 1.0f / total;
                if (live && a.shares > 1)
                    a.part.stats[share * a.part.rows + query_at(r)] = whole ? make_float2(0.0f, kWritten) : make_float2(m == -INFINITY ? m : shift, total);
                unsigned noted[8], any = 0u;
#pragma unroll
                for (int i = 0; i < 8; ++i) any |= noted[i] = lds_volatile_u32(base + Z::kNoted + 4 * i);
                auto add_noted = [&](uint32_t (&o)[32], int d) {
                    for (int i = 0; i < 8; ++i)
                        for (unsigned w = noted[i]; w; w &= w - 1) {
                            const int row = fewest + 32 * i + __ffs(w) - 1;
                            if (!live || row >= limit || row < start) continue;
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) + not_finite<T, false>(a, table, row, h, d + e));
                        }
                };
                // by way of the queries' place, 256 bytes of a row at a time (128 with 64 features), so that rows are written whole
                constexpr int PASS = D == 64 ? 128 : 256, LANES = PASS / 16, ROWS = 128 / LANES;
                uint8_t* const place = smem + t * Z::kQTile;
                const int mine = threadIdx.x & 127;
                auto through = [&](auto fill, char* to, int64_t row_bytes, int passes) {
                    for (int pass = 0; pass < passes; ++pass) {
                        fill(pass, place + mine * PASS);
                        role_barrier(t + 1, 128);
                        const int piece = mine % LANES;
#pragma unroll 8
                        for (int i = 0; i < 128 / ROWS; ++i) {
                            const int row = mine / LANES + i * ROWS;
                            if (t * kTileRows + row >= qt.rows) break;
                            const uint4 v = *reinterpret_cast<const uint4*>(place + row * PASS + ((piece ^ (row & 7)) << 4));
                            *reinterpret_cast<uint4*>(to + query_at(t * kTileRows + row) * row_bytes + pass * PASS + piece * 16) = v;
                        }
                        role_barrier(t + 1, 128);
                    }
                };
                if (whole) {
                    through([&](int pass, uint8_t* row) {
#pragma unroll
                        for (int d = 0; d < PASS / 2; d += 32) {
                            uint32_t o[32];
                            tmem_ld32(out + (uint32_t)(pass * (PASS / 2) + d), o);
                            tmem_wait_ld();
                            if (any) add_noted(o, pass * (PASS / 2) + d);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) w[e] = F16Bits<T>::pack(__uint_as_float(o[8 * i + 2 * e]) * inv, __uint_as_float(o[8 * i + 2 * e + 1]) * inv);
                                *reinterpret_cast<uint4*>(row + (((d / 8 + i) ^ (mine & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                    }, static_cast<char*>(a.out), D * 2, D * 2 / PASS);
                } else {
                    through([&](int pass, uint8_t* row) {
#pragma unroll
                        for (int d = 0; d < PASS / 4; d += 32) {
                            uint32_t o[32];
                            tmem_ld32(out + (uint32_t)(pass * (PASS / 4) + d), o);
                            tmem_wait_ld();
                            if (any) add_noted(o, pass * (PASS / 4) + d);
#pragma unroll
                            for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(row + (((d / 4 + i) ^ (mine & 7)) << 4)) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                        }
                    }, reinterpret_cast<char*>(a.part.sums + share * a.part.rows * D), D * 4, D * 4 / PASS);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem, Z::kColumns);
    }
}

int make_page_map(CUtensorMap* map, const void* ptr, int dt, const bi8_paged_cache& c, int64_t page, int64_t head, int64_t row, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return fail(BI8_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    ensure_current_context();
    const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.page_rows, (cuuint64_t)c.heads, (cuuint64_t)c.pages};
    // a dimension of one element needs no step, but the encoder wants one
    const cuuint64_t dense = (cuuint64_t)c.head_dim * 2;
    const cuuint64_t steps[3] = {(cuuint64_t)row * 2, c.heads > 1 ? (cuuint64_t)head * 2 : dense, c.pages > 1 ? (cuuint64_t)page * 2 : dense};
    const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1}, one[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, dt == BI8_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(ptr), dims, steps, box, one,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(BI8_ERR_CUDA, "cuTensorMapEncodeTiled (pages) failed with CUresult %d", (int)r);
    return BI8_OK;
}

template <typename T, int D>
int launch(const PagedAttnArgs& a, int dt, cudaStream_t st) {
    using Z = Shape<D>;
    int box_rows = 16;                                        // the largest power of two that divides a page, up to a step
    while (box_rows < Z::kRows && a.cache.page_rows % (2 * box_rows) == 0) box_rows *= 2;
    CUtensorMap k_map, v_map;
    if (int rc = make_page_map(&k_map, a.cache.k, dt, a.cache, a.cache.k_page, a.cache.k_head, a.cache.k_row, box_rows)) return rc;
    if (int rc = make_page_map(&v_map, a.cache.v, dt, a.cache, a.cache.v_page, a.cache.v_head, a.cache.v_row, box_rows)) return rc;
    if constexpr (Z::kTiles == 2) {
        // The roles' shares of the registers come out of what the block was launched with; were that less, their wait for it would not end.
        static std::atomic<int> registers{0};
        int n = registers.load(std::memory_order_relaxed);
        if (n == 0) {
            cudaFuncAttributes at;
            BI8_CUDA_TRY(cudaFuncGetAttributes(&at, paged_many_kernel<T, D>));
            registers.store(n = at.numRegs, std::memory_order_relaxed);
        }
        if (n * Z::kThreads < 128 * (2 * kSoftmaxRegisters + kOtherRegisters))
            return fail(BI8_ERR_CUDA, "attention_paged: built with %d registers a thread, too few for the kernel's roles", n);
    }
    int* const status = device_status_ptr();
    if (!status) return fail(BI8_ERR_CUDA, "attention_paged: the device's status word cannot be reached");
    static SmemOptIn opt_in;
    if (int rc = opt_in.ensure(paged_many_kernel<T, D>, Z::kBytes)) return rc;
    return launch_chained(paged_many_kernel<T, D>, (unsigned)((int64_t)a.tiles * a.Hkv * a.shares), Z::kThreads, Z::kBytes, st, k_map, v_map, a, box_rows, kShareRows, status,
                          4000000000ll);
}

}  // namespace

int paged_many_tile(int64_t D) { return D == 256 ? Shape<256>::kTiles * kTileRows : Shape<128>::kTiles * kTileRows; }

int launch_paged_many(const PagedAttnArgs& a, int dt, int64_t D, cudaStream_t st) {
    auto go = [&](auto* tag) {
        using E = std::remove_pointer_t<decltype(tag)>;
        if (D == 64) return launch<E, 64>(a, dt, st);
        if (D == 128) return launch<E, 128>(a, dt, st);
        return launch<E, 256>(a, dt, st);
    };
    return dt == BI8_BF16 ? go(static_cast<__nv_bfloat16*>(nullptr)) : go(static_cast<__half*>(nullptr));
}

}  // namespace bi8
