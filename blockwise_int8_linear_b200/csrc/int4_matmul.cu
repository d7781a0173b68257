// y = x W^T for a few rows of x and weights held in 4-bit blocks:
//   y[m, n] = sum_j s[n, j] / 7 * sum_{k in block j} q[n, k] x[m, k]  (+ bias[n]) (+ residual[m, n]),   fp32, rounded once.
//
// What bounds it is the weights: 4 bits of code and a sixteenth of a scale's bytes each, read once.  The sums run on the tensor cores
// with the codes as the 16-row operand and up to 64 rows of x as columns: unpacking a weight is one instruction (int4_common.cuh), and the
// columns that few rows of x leave empty cost nothing that counts.  (On the CUDA cores a weight takes an unpack, a conversion and a multiply-add per row of x: at 6.5 TB/s, 12 weights per
// ns, the SMs have three instructions for each.)
//
// A CTA of 16 warps, one an SM, keeps its share of x in shared memory, in the order of the codes, and goes through tiles of W: its warps are
// over rows (16 each) and over K, in pieces of 256 values (128 bytes a row), which come into the warp's ring of shared memory by
// asynchronous copies while an earlier one is multiplied.  CTAs of a cluster share the rows and divide K once more.  The sums of
// several tiles are collected before they are added, over the warps and over the cluster, in a fixed order: no workspace, no atomics, the
// same bits on every call.
//
// Measured, launched from a graph: one row through 4096 x 4096 6.0 us, 4096 -> 32000 19 us (3.65 TB/s); 8 rows through 4096 -> 11008 12 us,
// 16 17 us, 32 28 us, 64 50 us.  Few rows are bound by a warp's 580 instructions a piece (180 unpack, 230 more are the rest of the loop, the
// others fills, x and sums; IPC 2.1), small layers by latency.  Instances of 16 and more columns spill (12 to 92 bytes a thread at 16, 60 to 128 at
// 32, 220 to 460 at 64): 128 registers are what 512 threads have.
#include "int4_common.cuh"

#include <cooperative_groups.h>

#include <atomic>
#include <type_traits>

namespace bi8 {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 16, kThreads = kWarps * 32;
constexpr int kPiece = 256;                  // values of K that a warp takes at a time
constexpr int kSmemSM = 227 * 1024;          // shared memory that an SM's CTAs have

struct MatmulArgs {
    const void* x;
    int64_t ldx;
    const uint8_t* W;
    int64_t ldw;
    const unsigned short* sW;
    int64_t blocks;          // scales per row of W
    const void* bias;
    const void* residual;
    int64_t ldr;
    void* C;
    int64_t ldc;
    int bias_dtype, out_dtype;
    int M, N, K;
    int tiles;               // of 16 * warps_n rows of W
    int group;               // tiles whose sums a CTA collects before they are added
    int warps_n;             // warps of a CTA over rows of W; the others divide K
    int pieces;              // of K
    int ranks;               // CTAs of a cluster
    int pieces_cta;          // a CTA's share
    int pieces_stage;        // as many of them as x has room for
    bool x_vec, w_vec, s_vec;
};

__device__ __forceinline__ float load_as_float(const void* p, int dt, int64_t i) {
    if (dt == BI8_F32) return static_cast<const float*>(p)[i];
    if (dt == BI8_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_from_float(void* p, int dt, int64_t i, float y) {
    if (dt == BI8_F32) static_cast<float*>(p)[i] = y;
    else if (dt == BI8_F16) static_cast<__half*>(p)[i] = __float2half_rn(y);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(y);
}

// 32 bits of codes from any byte address: the two aligned words that hold them, each read only where it holds a byte before `end`.
__device__ __forceinline__ uint32_t load_word(const uint8_t* p, const uint8_t* end) {
    if (p >= end) return 0u;
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    const uint32_t* base = reinterpret_cast<const uint32_t*>(a & ~(uintptr_t)3);
    const uint32_t lo = __ldg(base);
    const uint32_t hi = reinterpret_cast<const uint8_t*>(base + 1) < end && (a & 3u) ? __ldg(base + 1) : 0u;
    return __funnelshift_r(lo, hi, (uint32_t)(a & 3u) * 8u);
}

// A warp's ring of pieces in shared memory: 16 rows of 128 bytes of codes, 32 bytes apart modulo 128 (the eight bytes that the lanes of
// four rows read are in different banks), then the rows' scales.
constexpr int kCodePitch = kPiece / 2 + 32;
template <int BLOCK>
constexpr int kPieceBytes = 16 * kCodePitch + 16 * (kPiece / BLOCK) * 2;

// One piece of 16 rows from `n0` on into shared memory.  Rows behind the last one are read as the last one (and not stored); codes behind a
// row's end are zero bytes, scales whatever (x is zero there).
template <int BLOCK>
__device__ __forceinline__ void fill(uint8_t* dst, const MatmulArgs& a, int n0, int piece, int lane) {
    constexpr int PER = kPiece / BLOCK;
    const int64_t at = (int64_t)piece * (kPiece / 2) + 16 * (lane & 7), kb = ((int64_t)a.K + 1) / 2;
    const int room = (int)max((int64_t)0, min((int64_t)16, kb - at));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = (lane >> 3) + 4 * i;
        const uint8_t* src = a.W + (int64_t)min(n0 + row, a.N - 1) * a.ldw;
        uint8_t* to = dst + row * kCodePitch + 16 * (lane & 7);
        if (a.w_vec) {
            copy16((uint32_t)__cvta_generic_to_shared(to), room > 0 ? src + at : src, room);
        } else {
            const uint8_t *from = src + at, *end = src + kb;
            *reinterpret_cast<uint4*>(to) = make_uint4(load_word(from, end), load_word(from + 4, end), load_word(from + 8, end), load_word(from + 12, end));
        }
    }
    if (lane < 16) {
        const int64_t j = (int64_t)piece * PER;
        const unsigned short* src = a.sW + (int64_t)min(n0 + lane, a.N - 1) * a.blocks + j;
        uint8_t* to = dst + 16 * kCodePitch + lane * (2 * PER);
        if (a.s_vec && j + PER <= a.blocks) {
            copy_some<2 * PER>((uint32_t)__cvta_generic_to_shared(to), src);
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) reinterpret_cast<unsigned short*>(to)[i] = j + i < a.blocks ? __ldg(src + i) : (unsigned short)0;
        }
    }
}

// Pieces of a warp in shared memory: one in use, the others on their way.
template <int NT>
constexpr int kRing = NT <= 2 ? 3 : 2;

// Sizes in shared memory: the warps' rings, x, and for a group of tiles the sums of the warps that share rows, with the CTA's own behind
// them where a cluster adds them.
template <int BLOCK, int NT>
constexpr int kRingBytes = kWarps * kRing<NT> * kPieceBytes<BLOCK>;
inline __host__ __device__ int x_pitch(int pieces) { return pieces * kPiece * 2 + 16; }
inline __host__ __device__ int sum_parts(int warps_k, int ranks) { return warps_k == 1 || ranks == 1 ? warps_k : warps_k + 1; }

template <typename T, int BLOCK, int NT>
__global__ void __launch_bounds__(kThreads, 1) matmul_int4_kernel(const MatmulArgs a) {
    constexpr int COLS = 8 * NT, PER = kPiece / BLOCK, RING = kRing<NT>;
    extern __shared__ __align__(16) uint8_t smem[];
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = a.ranks, rank = (int)(blockIdx.x % ranks);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int warps_k = kWarps / a.warps_n, wn = warp % a.warps_n, wk = warp / a.warps_n, rows_cta = 16 * a.warps_n;
    const int m0 = blockIdx.y * COLS, rows_x = min(COLS, a.M - m0);
    const int first = rank * a.pieces_cta, last = min(a.pieces, first + a.pieces_cta);
    const int tile_step = (int)(gridDim.x / ranks), tile0 = (int)(blockIdx.x / ranks);
    uint8_t* const ring = smem + warp * (RING * kPieceBytes<BLOCK>);
    // x: rows 16 bytes apart modulo 128, so that the lanes of two rows read different banks
    const int pitch = x_pitch(a.pieces_stage);
    uint8_t* const xs = smem + kRingBytes<BLOCK, NT>;
    const int sums = rows_x * rows_cta;
    float* const part = reinterpret_cast<float*>(xs + rows_x * pitch);       // [tile of the group][part][rows_x][rows_cta]

    // x of pieces base to end: as copies into the slots that the lanes read (lane c reads 32 bytes of every 64 values: what meets its two
    // words of codes; with blocks of 32, of both halves), then, by the thread that copied them, into the order of the codes.
    auto each_eight = [&](int base, int end, auto body) {
        if (base >= end) return;                              // a rank behind the last piece
        const int per_row = (end - base) * (kPiece / 8);
        int m = 0, p = threadIdx.x;
        while (true) {
            while (p >= per_row) p -= per_row, ++m;
            if (m >= rows_x) break;
            const int i = p & 7, slot = BLOCK == 32 ? (i & 3) * 2 + (i >> 2) : i;
            body(m, base * kPiece + 8 * p, xs + m * pitch + (p >> 3) * 128 + slot * 16);
            p += kThreads;
        }
    };
    auto fetch_x = [&](int base, int end) {
        each_eight(base, end, [&](int m, int k, uint8_t* to) {
            const unsigned short* src = static_cast<const unsigned short*>(a.x) + (int64_t)(m0 + m) * a.ldx;
            const int room = max(0, min(8, a.K - k));
            if (a.x_vec) {
                copy16((uint32_t)__cvta_generic_to_shared(to), room > 0 ? src + k : src, 2 * room);
            } else {
                uint32_t e[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = j < room ? __ldg(src + k + j) : 0u;
                *reinterpret_cast<uint4*>(to) = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
            }
        });
    };
    auto order_x = [&](int base, int end) {
        each_eight(base, end, [&](int, int, uint8_t* at) {
            uint4* p = reinterpret_cast<uint4*>(at);
            *p = paired8(*p);
        });
    };

    after_predecessor();
    const bool once = a.pieces_cta <= a.pieces_stage;         // all of this CTA's x fits
    if (once) fetch_x(first, last);
    commit_copies();
    // What is filled next: a tile and a piece of it, and this lane's part: 16 bytes of every fourth row, a row's scales.  The addresses move
    // on by constants; they are used where the piece is whole and aligned and all of its rows exist.
    int f_tile = tile0, f_piece = first + wk, in = 0, out = 0;
    const int aligned_pieces = a.w_vec && a.s_vec ? a.K / kPiece : 0, whole_tiles = a.N / rows_cta;
    const int64_t row0 = (int64_t)tile0 * rows_cta + 16 * wn;
    const uint8_t* w_tile = a.W + (row0 + (lane >> 3)) * a.ldw + (int64_t)f_piece * (kPiece / 2) + 16 * (lane & 7);
    const unsigned short* s_tile = a.sW + (row0 + (lane & 15)) * a.blocks + (int64_t)f_piece * PER;
    const int64_t w_tile_step = (int64_t)tile_step * rows_cta * a.ldw, s_tile_step = (int64_t)tile_step * rows_cta * a.blocks, w_rows = 4 * a.ldw;
    const uint8_t* w_at = w_tile;
    const unsigned short* s_at = s_tile;
    const uint32_t w_slot = (uint32_t)__cvta_generic_to_shared(ring + (lane >> 3) * kCodePitch + 16 * (lane & 7));
    const uint32_t s_slot = (uint32_t)__cvta_generic_to_shared(ring + 16 * kCodePitch + (lane & 15) * (2 * PER));
    auto fill_next = [&] {
        if (f_piece >= last) {
            f_piece = first + wk, f_tile += tile_step;
            w_at = w_tile += w_tile_step;
            s_at = s_tile += s_tile_step;
        }
        if (f_tile < a.tiles && f_piece < last) {
            if (f_piece < aligned_pieces && f_tile < whole_tiles) {
                const uint32_t to = w_slot + in * kPieceBytes<BLOCK>;
                const uint8_t* src = w_at;
#pragma unroll
                for (int i = 0; i < 4; ++i, src += w_rows) copy16(to + 4 * i * kCodePitch, src);
                if (lane < 16) copy_some<2 * PER>(s_slot + in * kPieceBytes<BLOCK>, s_at);
            } else {
                fill<BLOCK>(ring + in * kPieceBytes<BLOCK>, a, f_tile * rows_cta + 16 * wn, f_piece, lane);
            }
        }
        commit_copies();
        f_piece += warps_k;
        w_at += warps_k * (kPiece / 2);
        s_at += warps_k * PER;
        in = in + 1 == RING ? 0 : in + 1;
    };
#pragma unroll
    for (int i = 0; i < RING - 1; ++i) fill_next();
    if (once) {
        wait_copies<RING - 1>();
        order_x(first, last);
        __syncthreads();
    }

    const int parts = sum_parts(warps_k, ranks);
    for (int group = tile0; group < a.tiles; group += a.group * tile_step) {
        // ---- the group's tiles one after the other; no warp waits for another one in between
        const int count = min(a.group, (a.tiles - group + tile_step - 1) / tile_step);
        for (int in_group = 0; in_group < count; ++in_group) {
            float y[NT][4] = {};
            for (int base = first, piece = first + wk; base < last; base += a.pieces_stage) {
                const int end = min(last, base + a.pieces_stage);
                if (!once) {
                    __syncthreads();
                    fetch_x(base, end);
                    commit_copies();
                    wait_copies<0>();
                    order_x(base, end);
                    __syncthreads();
                }
                for (; piece < end; piece += warps_k) {
                    fill_next();                                  // into the slot that every lane left at the end of the piece before
                    wait_copies<RING - 1>();
                    __syncwarp();
                    const uint8_t* const lo = ring + out * kPieceBytes<BLOCK> + g * kCodePitch + (BLOCK == 32 ? 4 : 8) * c;
                    const uint8_t* const hi = lo + 8 * kCodePitch;
                    const uint32_t* const sp = reinterpret_cast<const uint32_t*>(ring + out * kPieceBytes<BLOCK> + 16 * kCodePitch + g * (2 * PER));
                    uint32_t sw[2][PER / 2];
#pragma unroll
                    for (int i = 0; i < PER / 2; ++i) sw[0][i] = sp[i], sw[1][i] = sp[4 * PER + i];
                    auto scale = [&](int r, int i) { return i & 1 ? F16Bits<T>::hi(sw[r][i / 2]) : F16Bits<T>::lo(sw[r][i / 2]); };
                    const uint8_t* const xp = xs + (piece - base) * (kPiece * 2) + c * 32;
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        uint2 w0, w1;
                        if (BLOCK == 32) {
                            w0 = make_uint2(*reinterpret_cast<const uint32_t*>(lo + 32 * u), *reinterpret_cast<const uint32_t*>(lo + 32 * u + 16));
                            w1 = make_uint2(*reinterpret_cast<const uint32_t*>(hi + 32 * u), *reinterpret_cast<const uint32_t*>(hi + 32 * u + 16));
                        } else {
                            w0 = *reinterpret_cast<const uint2*>(lo + 32 * u);
                            w1 = *reinterpret_cast<const uint2*>(hi + 32 * u);
                        }
                        const Codes4 r0a = unpack8<T>(w0.x), r0b = unpack8<T>(w0.y), r1a = unpack8<T>(w1.x), r1b = unpack8<T>(w1.y);
                        const int AFTER = BLOCK == 32 ? 2 * u + 1 : u * PER / 4;         // the scale of (the second half of) these 64 values
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            // columns behind the last row of x read that row again and are not stored
                            const uint4* p = reinterpret_cast<const uint4*>(xp + min(8 * t + g, rows_x - 1) * pitch + u * 128);
                            const uint4 xa = p[0], xb = p[1];
                            auto scaled = [&](const float (&d)[4], int i) {
                                y[t][0] = fmaf(d[0], scale(0, i), y[t][0]);
                                y[t][1] = fmaf(d[1], scale(0, i), y[t][1]);
                                y[t][2] = fmaf(d[2], scale(1, i), y[t][2]);
                                y[t][3] = fmaf(d[3], scale(1, i), y[t][3]);
                            };
                            float d[4];
                            mma16_first<T>(d, r0a.p04, r1a.p04, r0a.p15, r1a.p15, xa.x, xa.y);
                            mma16<T>(d, r0a.p26, r1a.p26, r0a.p37, r1a.p37, xa.z, xa.w);
                            if (BLOCK == 32) {
                                scaled(d, 2 * u);
                                mma16_first<T>(d, r0b.p04, r1b.p04, r0b.p15, r1b.p15, xb.x, xb.y);
                            } else {
                                mma16<T>(d, r0b.p04, r1b.p04, r0b.p15, r1b.p15, xb.x, xb.y);
                            }
                            mma16<T>(d, r0b.p26, r1b.p26, r0b.p37, r1b.p37, xb.z, xb.w);
                            scaled(d, AFTER);
                        }
                    }
                    out = out + 1 == RING ? 0 : out + 1;
                    __syncwarp();
                }
            }
            float* const mine = part + (size_t)(in_group * parts + wk) * sums;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int col = 8 * t + 2 * c + (i & 1);
                    if (col < rows_x) mine[col * rows_cta + 16 * wn + g + 8 * (i >> 1)] = y[t][i];
                }
        }
        __syncthreads();
        // ---- sums over the warps that share rows, then over the cluster: both in a fixed order.  Four rows at a time; loads are under way
        // before the first sum.
        auto add = [](float4& s, const float4& v) { s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w; };
        auto warps_sum = [&](const float* p) {
            float4 s = *reinterpret_cast<const float4*>(p);
            for (int w0 = 1; w0 < warps_k; w0 += 3) {             // 2, 4, 8 or 16 warps: 1, 3, 7 or 15 more
                float4 v[3];
#pragma unroll
                for (int w = 0; w < 3; ++w)
                    if (w0 + w < warps_k) v[w] = *reinterpret_cast<const float4*>(p + (size_t)(w0 + w) * sums);
#pragma unroll
                for (int w = 0; w < 3; ++w)
                    if (w0 + w < warps_k) add(s, v[w]);
            }
            return s;
        };
        auto store = [&](int tile, int i, const float4& s) {
            const int m = m0 + i / rows_cta, n = tile * rows_cta + i % rows_cta;
            const float y[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (n + j >= a.N) return;
                float v = y[j] * (1.0f / 7.0f / kCodeUnit<T>);
                if (a.bias) v += load_as_float(a.bias, a.bias_dtype, n + j);
                if (a.residual) v += load_as_float(a.residual, a.out_dtype, (int64_t)m * a.ldr + n + j);
                store_from_float(a.C, a.out_dtype, (int64_t)m * a.ldc + n + j, v);
            }
        };
        const int values = count * sums;
        if (ranks == 1) {
            for (int i = 4 * threadIdx.x; i < values; i += 4 * kThreads) {
                const int k = i / sums, e = i - k * sums;
                store(group + k * tile_step, e, warps_sum(part + (size_t)k * parts * sums + e));
            }
        } else {
            if (warps_k > 1)
                for (int i = 4 * threadIdx.x; i < values; i += 4 * kThreads) {
                    const int k = i / sums, e = i - k * sums;
                    float* const p = part + (size_t)k * parts * sums + e;
                    *reinterpret_cast<float4*>(p + (size_t)warps_k * sums) = warps_sum(p);
                }
            cluster.sync();
            const int share = (values / 4 + ranks - 1) / ranks * 4;
            for (int i = rank * share + 4 * threadIdx.x; i < min(values, (rank + 1) * share); i += 4 * kThreads) {
                const int k = i / sums, e = i - k * sums;
                float* const p = part + (size_t)(k * parts + parts - 1) * sums + e;
                float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (int r0 = 0; r0 < ranks; r0 += 4) {
                    float4 v[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (r0 + r < ranks) v[r] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(p, r0 + r));
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (r0 + r < ranks) add(s, v[r]);
                }
                store(group + k * tile_step, e, s);
            }
        }
        if (group + a.group * tile_step < a.tiles) {              // the next group overwrites what the others read
            if (ranks > 1) cluster.sync();
            else __syncthreads();
        }
    }
    wait_copies<0>();
    if (ranks > 1) cluster.sync();           // the others read this CTA's sums
}

// How a product is divided: a CTA's warps over rows of W (the others divide its K), the CTAs of a cluster over K.
struct Division {
    int warps_n, ranks, pieces_cta, pieces_stage, tiles, group, grid;
    size_t smem;
    double cost;
};

template <typename T, int BLOCK, int NT>
int launch(MatmulArgs a, cudaStream_t st) {
    constexpr int COLS = 8 * NT;
    static SmemOptIn opt_in;
    const int m_tiles = (a.M + COLS - 1) / COLS, rows_x = a.M < COLS ? a.M : COLS, sms = sm_count();
    a.pieces = (a.K + kPiece - 1) / kPiece;
    // The division with the shortest estimate, in cycles.  An SM has one CTA, which goes through its tiles one after the other: its warps
    // take a piece in the time that their matrix and other instructions need, or, if it is their only one, in one piece's latency.
    // clusters of 1, 2, 4 and 8 such CTAs that the device runs at once: fewer than its SMs would hold, which come in groups
    static std::atomic<int> at_once[64][4];
    int dev = 0;
    BI8_CUDA_TRY(current_device(&dev));
    if (dev < 0 || dev >= 64) return fail(BI8_ERR_CUDA, "device ordinal %d out of range", dev);
    if (int rc = opt_in.ensure(matmul_int4_kernel<T, BLOCK, NT>, kSmemSM - 1024)) return rc;
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(kThreads);
    cfg.attrs = attr;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    for (int r = 0; r < 4; ++r) {
        if (at_once[dev][r].load(std::memory_order_relaxed) > 0) continue;
        int n = 0;
        attr[0].val.clusterDim.x = 1u << r;
        cfg.gridDim = dim3((unsigned)sms / 8 * 8);
        cfg.dynamicSmemBytes = kSmemSM - 1024;
        cfg.numAttrs = 1;
        BI8_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, matmul_int4_kernel<T, BLOCK, NT>, &cfg));
        at_once[dev][r].store(n > 0 ? n : 1, std::memory_order_relaxed);
    }
    Division best{};
    best.cost = 1e30;
    auto consider = [&](int wn, int ranks) {
        const int wk = kWarps / wn, cta = (a.pieces + ranks - 1) / ranks, tiles = (a.N + 16 * wn - 1) / (16 * wn);
        const size_t sums = (size_t)sum_parts(wk, ranks) * rows_x * 16 * wn * 4, fixed = kRingBytes<BLOCK, NT> + sums, limit = kSmemSM - 1024;
        if (fixed + (size_t)rows_x * x_pitch(1) > limit) return;
        int stage = cta;
        if (fixed + (size_t)rows_x * x_pitch(stage) > limit) stage = ((int)((limit - fixed) / rows_x) - 16) / (kPiece * 2);
        const int room = at_once[dev][ranks == 1 ? 0 : ranks == 2 ? 1 : ranks == 4 ? 2 : 3].load(std::memory_order_relaxed);
        int clusters = room / m_tiles;
        if (clusters < 1) clusters = 1;
        if (clusters > tiles) clusters = tiles;
        const int rounds = (tiles + clusters - 1) / clusters;
        clusters = (tiles + rounds - 1) / rounds;
        size_t bytes = fixed + (size_t)rows_x * x_pitch(stage);
        int group = (int)((limit - bytes) / sums) + 1;
        if (group > rounds) group = rounds;
        group = (rounds + (rounds + group - 1) / group - 1) / ((rounds + group - 1) / group);
        bytes += (group - 1) * sums;
        const double waves = ((int64_t)clusters * m_tiles + room - 1) / room, pieces = (cta + wk - 1) / wk;
        // a tile: its pieces on all warps, x again where it does not stay, what is left of the loop; x, once; a group's sums, over
        // the warps and then over the cluster, each of whose CTAs stores its share (taking 16 rows through 4096 -> 11008 from 21 us to 17)
        const double tile = pieces * kWarps * (110.0 + 50.0 * NT) + (stage < cta ? 30.0 * rows_x * cta + 2000.0 * ((cta + stage - 1) / stage) : 0.0) + 450.0;
        const double quads = (double)group * rows_x * wn * 4 / kThreads;
        const double reduction = 600.0 + (wk > 1 ? quads * (300.0 + 80.0 * wk) : 0.0) + quads / ranks * 1500.0 + (ranks > 1 ? 600.0 + 700.0 * ranks : 0.0);
        const double cost = waves * (4000.0 + 30.0 * rows_x * cta + rounds * tile + (rounds + group - 1) / group * reduction);
        if (cost < best.cost) best = {wn, ranks, cta, stage, tiles, group, clusters * ranks, bytes, cost};
    };
    for (int wn = 1; wn <= kWarps; wn *= 2)
        for (int ranks = 1; ranks <= 8; ranks *= 2)
            if (ranks == 1 || a.pieces >= ranks) consider(wn, ranks);
    a.warps_n = best.warps_n, a.ranks = best.ranks, a.pieces_cta = best.pieces_cta, a.pieces_stage = best.pieces_stage, a.tiles = best.tiles, a.group = best.group;
    cfg.gridDim = dim3((unsigned)best.grid, (unsigned)m_tiles);
    cfg.dynamicSmemBytes = best.smem;
    cfg.stream = st;
    attr[0].val.clusterDim.x = (unsigned)best.ranks;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
    BI8_CUDA_TRY(cudaLaunchKernelEx(&cfg, matmul_int4_kernel<T, BLOCK, NT>, a));
    return BI8_OK;
}

}  // namespace

int launch_matmul_int4(const void* x, int x_dt, int64_t ldx, const uint8_t* W, int64_t ldw, const void* sW, const void* bias, int bias_dt,
                       const void* residual, int64_t ldr, void* C, int64_t ldc, int out_dt, int64_t M, int64_t N, int64_t K, int block,
                       cudaStream_t st) {
    MatmulArgs a{};
    a.x = x;
    a.ldx = ldx;
    a.W = W;
    a.ldw = ldw;
    a.sW = static_cast<const unsigned short*>(sW);
    a.blocks = (K + block - 1) / block;
    a.bias = bias;
    a.residual = residual;
    a.ldr = ldr;
    a.C = C;
    a.ldc = ldc;
    a.bias_dtype = bias_dt;
    a.out_dtype = out_dt;
    a.M = (int)M;
    a.N = (int)N;
    a.K = (int)K;
    a.x_vec = aligned(x, 16) && (M == 1 || ldx % 8 == 0);
    a.w_vec = aligned(W, 16) && (N == 1 || ldw % 16 == 0);
    const int scale_bytes = 2 * kPiece / block;
    a.s_vec = aligned(sW, scale_bytes) && (N == 1 || a.blocks % (kPiece / block) == 0);
    auto by_columns = [&](auto* tag, auto blk) {
        using T = std::remove_pointer_t<decltype(tag)>;
        constexpr int B = decltype(blk)::value;
        if (M <= 8) return launch<T, B, 1>(a, st);
        if (M <= 16) return launch<T, B, 2>(a, st);
        if (M <= 32) return launch<T, B, 4>(a, st);
        return launch<T, B, 8>(a, st);
    };
    auto by_block = [&](auto* tag) {
        if (block == 32) return by_columns(tag, std::integral_constant<int, 32>{});
        if (block == 64) return by_columns(tag, std::integral_constant<int, 64>{});
        return by_columns(tag, std::integral_constant<int, 128>{});
    };
    return x_dt == BI8_BF16 ? by_block(static_cast<__nv_bfloat16*>(nullptr)) : by_block(static_cast<__half*>(nullptr));
}

}  // namespace bi8
