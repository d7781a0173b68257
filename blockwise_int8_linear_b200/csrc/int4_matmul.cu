// y = x W^T for a few rows of x and weights held in 4-bit blocks:
//   y[m, n] = sum_j s[n, j] / 7 * sum_{k in block j} q[n, k] x[m, k]  (+ bias[n]) (+ residual[m, n]),   fp32, rounded once.
//
// What bounds it is the weights: 4 bits of code and a sixteenth of a scale's bytes each, read once.  The sums run on the tensor cores
// with the codes as the 16-row operand and up to 64 rows of x as columns: unpacking a weight is one instruction (int4_common.cuh), and the
// columns that few rows of x leave empty cost nothing that counts.  (On the CUDA cores a weight takes an unpack, a conversion and a multiply-add per row of x: at 6.5 TB/s, 12 weights per
// ns, the SMs have three instructions for each.)
//
// A warp takes 16 rows of W and strides over K in pieces of 256 (128 bytes a row; lane 4g + c reads 8 bytes of rows g and g + 8 for every 64
// values), the next piece's loads in flight while this one is multiplied.  A CTA is eight warps, over rows and over K; CTAs of a
// cluster share the rows and divide K once more, and add what they have over distributed shared memory in rank order: no
// workspace, no atomics, the same bits on every call.  x comes through shared memory as fp16 with a power of two
// per row and 64 (32) values.
#include "int4_common.cuh"

#include <cooperative_groups.h>

#include <type_traits>

namespace bi8 {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kPiece = 256;                  // values of K that a warp takes at a time
constexpr int kMaxStage = 160 * 1024;        // shared memory for x

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
    int M, N;
    int64_t K;
    int shift;               // log2 of the block
    int warps_n;             // warps of a CTA over rows of W; the others divide K
    int pieces;              // of K
    int pieces_cta;          // a cluster rank's share
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

// One piece of 16 rows as a lane holds it: for each 64 values two words of row g and two of row g + 8, and the rows' scales.
struct Piece {
    uint2 w[2][4];
    uint32_t s[2][4];        // bits of the scale of each 64 values (SHORT: of both halves)
};

// SHORT: blocks of 32, a lane's two words of 64 values lie in the two blocks; else the eight bytes lie in one.
// VEC: code rows begin on 8-byte boundaries.
template <bool SHORT, bool VEC>
__device__ __forceinline__ void load_piece(Piece& p, const MatmulArgs& a, const uint8_t* const (&row)[2], const unsigned short* const (&srow)[2],
                                           int piece, int c) {
    const int64_t kb = (a.K + 1) / 2, at = (int64_t)piece * (kPiece / 2);
    const bool full = at + kPiece / 2 <= kb;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t o = at + 32 * u + (SHORT ? 4 : 8) * c;
            if (VEC && !SHORT) {
                p.w[r][u] = make_uint2(0u, 0u);
                if (full || o < kb) p.w[r][u] = __ldg(reinterpret_cast<const uint2*>(row[r] + o));
            } else if (VEC) {
                p.w[r][u] = make_uint2(0u, 0u);
                if (full || o < kb) p.w[r][u].x = __ldg(reinterpret_cast<const uint32_t*>(row[r] + o));
                if (full || o + 16 < kb) p.w[r][u].y = __ldg(reinterpret_cast<const uint32_t*>(row[r] + o + 16));
            } else {
                p.w[r][u] = make_uint2(load_word(row[r] + o, row[r] + kb), load_word(row[r] + o + (SHORT ? 16 : 4), row[r] + kb));
            }
        }
        // scales: four, two or eight neighbouring ones
        const int64_t j = (int64_t)piece * kPiece >> a.shift;
        if (a.s_vec && full) {
            if (SHORT) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(srow[r] + j));
                p.s[r][0] = v.x, p.s[r][1] = v.y, p.s[r][2] = v.z, p.s[r][3] = v.w;
            } else if (a.shift == 6) {
                const uint2 v = __ldg(reinterpret_cast<const uint2*>(srow[r] + j));
                p.s[r][0] = v.x & 0xffffu, p.s[r][1] = v.x >> 16, p.s[r][2] = v.y & 0xffffu, p.s[r][3] = v.y >> 16;
            } else {
                const uint32_t v = __ldg(reinterpret_cast<const uint32_t*>(srow[r] + j));
                p.s[r][0] = p.s[r][1] = v & 0xffffu, p.s[r][2] = p.s[r][3] = v >> 16;
            }
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t i = ((int64_t)piece * kPiece + 64 * u) >> a.shift;
                uint32_t v = i < a.blocks ? (uint32_t)__ldg(srow[r] + i) : 0u;
                if (SHORT && i + 1 < a.blocks) v |= (uint32_t)__ldg(srow[r] + i + 1) << 16;
                p.s[r][u] = v;
            }
        }
    }
}

template <typename T, bool SHORT, int NT, bool VEC>
__global__ void __launch_bounds__(kThreads) matmul_int4_kernel(const MatmulArgs a) {
    constexpr int SEG = SHORT ? 32 : 64;     // values under one power of two of x
    constexpr int COLS = 8 * NT;
    extern __shared__ __align__(16) uint8_t smem[];
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int warps_k = kWarps / a.warps_n, wn = warp % a.warps_n, wk = warp / a.warps_n;
    const int m0 = blockIdx.y * COLS, rows_x = min(COLS, a.M - m0);
    const int n0 = (int)(blockIdx.x / ranks) * 16 * a.warps_n + 16 * wn;
    const int first = rank * a.pieces_cta, last = min(a.pieces, first + a.pieces_cta);
    const int stage = a.pieces_stage;
    // x: rows of `stage` pieces, 16 bytes apart modulo 128, so that the lanes of two rows read different banks; then the power of two of
    // every segment and column
    const int pitch = stage * kPiece * 2 + 16;
    uint8_t* const xs = smem;
    float* const seg = reinterpret_cast<float*>(smem + (size_t)rows_x * pitch);

    after_predecessor();
    const uint8_t* row[2];
    const unsigned short* srow[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int64_t n = min(n0 + g + 8 * r, a.N - 1);       // rows behind the last one read it again and are not stored
        row[r] = a.W + n * a.ldw;
        srow[r] = a.sW + n * a.blocks;
    }
    float y[NT][4] = {};
    Piece cur, nxt;
    int piece = first + wk;
    if (piece < last) load_piece<SHORT, VEC>(cur, a, row, srow, piece, c);

    for (int base = first; base < last; base += stage) {
        const int end = min(last, base + stage);
        if (base > first) __syncthreads();
        // ---- x into shared memory: a thread takes eight values, SEG / 8 lanes a segment
        const int per_row = (end - base) * (kPiece / 8);
        for (int i = threadIdx.x; i < rows_x * per_row; i += kThreads) {       // per_row is a multiple of 32: whole warps
            const int m = i / per_row, p = i - m * per_row;
            const int64_t k = (int64_t)base * kPiece + 8 * p;
            const unsigned short* src = static_cast<const unsigned short*>(a.x) + (int64_t)(m0 + m) * a.ldx + k;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (a.x_vec && k + 8 <= a.K) {
                v = __ldg(reinterpret_cast<const uint4*>(src));
            } else if (k < a.K) {
                uint32_t e[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = k + j < a.K ? __ldg(src + j) : 0u;
                v = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
            }
            uint32_t big = absmax8(v);
#pragma unroll
            for (int d = 1; d < SEG / 8; d <<= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, d));
            const float2 f = fit_fp16<T>(big);
            const uint4 o = operand8<T>(v, f.y);
            // lane c of a warp reads 32 bytes of every 64 values: what meets its two words of codes
            const int in = p & 7, slot = SHORT ? (in & 3) * 2 + (in >> 2) : in;
            *reinterpret_cast<uint4*>(xs + (size_t)m * pitch + (p >> 3) * 128 + slot * 16) = o;
            if ((p & (SEG / 8 - 1)) == 0) seg[(p / (SEG / 8)) * COLS + m] = f.x;
        }
        const int segs = (end - base) * (kPiece / SEG);
        if (rows_x < COLS)
            for (int i = threadIdx.x; i < segs * (COLS - rows_x); i += kThreads)
                seg[i / (COLS - rows_x) * COLS + rows_x + i % (COLS - rows_x)] = 0.0f;
        __syncthreads();

        // ---- this warp's pieces
        for (; piece < end; piece += warps_k) {
            const int next = piece + warps_k;
            if (next < last) load_piece<SHORT, VEC>(nxt, a, row, srow, next, c);
            const int u0 = (piece - base) * 4;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const Codes4 r0a = unpack8(cur.w[0][u].x), r0b = unpack8(cur.w[0][u].y);
                const Codes4 r1a = unpack8(cur.w[1][u].x), r1b = unpack8(cur.w[1][u].y);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    uint4 xa = make_uint4(0u, 0u, 0u, 0u), xb = xa;
                    if (8 * t + g < rows_x) {
                        const uint4* p = reinterpret_cast<const uint4*>(xs + (size_t)(8 * t + g) * pitch + (u0 + u) * 128 + c * 32);
                        xa = p[0];
                        xb = p[1];
                    }
                    const float* sp = seg + (size_t)(u0 + u) * (64 / SEG) * COLS + 8 * t + 2 * c;
                    const float2 f = *reinterpret_cast<const float2*>(sp);
                    float d[4] = {};
                    mma_f16(d, r0a.p04, r1a.p04, r0a.p15, r1a.p15, xa.x, xa.y);
                    mma_f16(d, r0a.p26, r1a.p26, r0a.p37, r1a.p37, xa.z, xa.w);
                    if (SHORT) {
                        const float s0 = F16Bits<T>::one(cur.s[0][u] & 0xffffu), s1 = F16Bits<T>::one(cur.s[1][u] & 0xffffu);
                        y[t][0] = fmaf(d[0], s0 * f.x, y[t][0]);
                        y[t][1] = fmaf(d[1], s0 * f.y, y[t][1]);
                        y[t][2] = fmaf(d[2], s1 * f.x, y[t][2]);
                        y[t][3] = fmaf(d[3], s1 * f.y, y[t][3]);
                        const float2 h = *reinterpret_cast<const float2*>(sp + COLS);
                        float e[4] = {};
                        mma_f16(e, r0b.p04, r1b.p04, r0b.p15, r1b.p15, xb.x, xb.y);
                        mma_f16(e, r0b.p26, r1b.p26, r0b.p37, r1b.p37, xb.z, xb.w);
                        const float t0 = F16Bits<T>::one(cur.s[0][u] >> 16), t1 = F16Bits<T>::one(cur.s[1][u] >> 16);
                        y[t][0] = fmaf(e[0], t0 * h.x, y[t][0]);
                        y[t][1] = fmaf(e[1], t0 * h.y, y[t][1]);
                        y[t][2] = fmaf(e[2], t1 * h.x, y[t][2]);
                        y[t][3] = fmaf(e[3], t1 * h.y, y[t][3]);
                    } else {
                        mma_f16(d, r0b.p04, r1b.p04, r0b.p15, r1b.p15, xb.x, xb.y);
                        mma_f16(d, r0b.p26, r1b.p26, r0b.p37, r1b.p37, xb.z, xb.w);
                        const float s0 = F16Bits<T>::one(cur.s[0][u]), s1 = F16Bits<T>::one(cur.s[1][u]);
                        y[t][0] = fmaf(d[0], s0 * f.x, y[t][0]);
                        y[t][1] = fmaf(d[1], s0 * f.y, y[t][1]);
                        y[t][2] = fmaf(d[2], s1 * f.x, y[t][2]);
                        y[t][3] = fmaf(d[3], s1 * f.y, y[t][3]);
                    }
                }
            }
            cur = nxt;
        }
    }

    // ---- sums over the warps that share rows, then over the cluster: both in a fixed order
    __syncthreads();
    const int rows_cta = 16 * a.warps_n;
    float* const part = reinterpret_cast<float*>(smem);                      // [warps_k][COLS][rows_cta]
    float* const total = part + (size_t)warps_k * COLS * rows_cta;           // [COLS][rows_cta]
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            part[((size_t)wk * COLS + 8 * t + 2 * c + (i & 1)) * rows_cta + 16 * wn + g + 8 * (i >> 1)] = y[t][i];
    __syncthreads();
    const int values = rows_x * rows_cta;
    for (int i = threadIdx.x; i < values; i += kThreads) {
        float s = part[i];
        for (int w = 1; w < warps_k; ++w) s += part[(size_t)w * COLS * rows_cta + i];
        total[i] = s;
    }
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    const int tile0 = (int)(blockIdx.x / ranks) * rows_cta;
    const int share = (values + ranks - 1) / ranks;
    for (int i = rank * share + threadIdx.x; i < min(values, (rank + 1) * share); i += kThreads) {
        float s = 0.0f;
        if (ranks == 1) s = total[i];
        else
            for (int r = 0; r < ranks; ++r) s += cluster.map_shared_rank(total, r)[i];
        const int m = m0 + i / rows_cta, n = tile0 + i % rows_cta;
        if (n >= a.N) continue;
        float out = s * (1.0f / 7.0f);
        if (a.bias) out += load_as_float(a.bias, a.bias_dtype, n);
        if (a.residual) out += load_as_float(a.residual, a.out_dtype, (int64_t)m * a.ldr + n);
        store_from_float(a.C, a.out_dtype, (int64_t)m * a.ldc + n, out);
    }
    if (ranks > 1) cluster.sync();           // the others read this CTA's sums
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

template <typename T, bool SHORT, int NT, bool VEC>
int launch(MatmulArgs a, cudaStream_t st) {
    constexpr int COLS = 8 * NT;
    static SmemOptIn opt_in;
    // Rows of W per CTA grow with the rows of x, which every CTA reads.
    a.warps_n = a.M <= 2 ? 1 : a.M <= 8 ? 2 : a.M <= 16 ? 4 : 8;
    const int tiles = (a.N + 16 * a.warps_n - 1) / (16 * a.warps_n), warps_k = kWarps / a.warps_n;
    const int m_tiles = (a.M + COLS - 1) / COLS;
    a.pieces = (int)((a.K + kPiece - 1) / kPiece);
    // CTAs of a cluster divide K until there are two CTAs an SM, as long as every warp keeps a piece.
    int ranks = 1;
    while (ranks < 8 && (int64_t)tiles * m_tiles * ranks < 2 * sm_count() && a.pieces >= 2 * ranks * warps_k) ranks *= 2;
    a.pieces_cta = (a.pieces + ranks - 1) / ranks;
    const int rows_x = a.M < COLS ? a.M : COLS;
    const int per_piece = rows_x * kPiece * 2 + (kPiece / (SHORT ? 32 : 64)) * COLS * 4;
    a.pieces_stage = a.pieces_cta;
    if ((int64_t)a.pieces_stage * per_piece + rows_x * 16 > kMaxStage) a.pieces_stage = (kMaxStage - rows_x * 16) / per_piece;
    size_t smem = (size_t)a.pieces_stage * per_piece + rows_x * 16;
    const size_t sums = (size_t)(warps_k + 1) * COLS * 16 * a.warps_n * 4;
    if (smem < sums) smem = sums;
    if (int rc = opt_in.ensure(matmul_int4_kernel<T, SHORT, NT, VEC>, smem)) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(tiles * ranks), (unsigned)m_tiles);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    BI8_CUDA_TRY(cudaLaunchKernelEx(&cfg, matmul_int4_kernel<T, SHORT, NT, VEC>, a));
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
    a.K = K;
    a.shift = block == 32 ? 5 : block == 64 ? 6 : 7;
    a.x_vec = aligned(x, 16) && (M == 1 || ldx % 8 == 0);
    a.w_vec = aligned(W, 8) && (N == 1 || ldw % 8 == 0);
    const int scale_bytes = 2 * kPiece / block;
    a.s_vec = aligned(sW, scale_bytes) && (N == 1 || a.blocks % (kPiece / block) == 0);
    auto by_columns = [&](auto* tag, auto is_short, auto vec) {
        using T = std::remove_pointer_t<decltype(tag)>;
        constexpr bool S = decltype(is_short)::value, V = decltype(vec)::value;
        if (M <= 8) return launch<T, S, 1, V>(a, st);
        if (M <= 16) return launch<T, S, 2, V>(a, st);
        if (M <= 32) return launch<T, S, 4, V>(a, st);
        return launch<T, S, 8, V>(a, st);
    };
    auto by_layout = [&](auto* tag, auto is_short) { return a.w_vec ? by_columns(tag, is_short, std::true_type{}) : by_columns(tag, is_short, std::false_type{}); };
    auto by_block = [&](auto* tag) { return block == 32 ? by_layout(tag, std::true_type{}) : by_layout(tag, std::false_type{}); };
    return x_dt == BI8_BF16 ? by_block(static_cast<__nv_bfloat16*>(nullptr)) : by_block(static_cast<__half*>(nullptr));
}

}  // namespace bi8
