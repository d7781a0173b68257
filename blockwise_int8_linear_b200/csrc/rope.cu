// Rotary positions of any tensor [B, T, H, D]: the first R features of every head are turned by the angles of the token's position
// (rope.cuh), the others copied.  The gradient is the same operation with the angles' signs changed (`conj`): the rotation's transpose.
//
// Bound by memory: x read once, the result written once, the table's rows from the caches.  A thread has its two pieces in kHeads heads of one token, so
// that a row of the table is read once for both, and all of its loads are under way before the first is used.  4 x 4096 tokens of 40 heads of
// 128 bf16 features: 58 us in a loop, 87 % of a copy's bandwidth.  (Four blocks an SM want 64 registers a thread: with four heads it spilled, 74 us a call
// alone against 61, and without that bound had too few loads under way, 68.)
#include "rope.cuh"

#include <type_traits>

namespace bi8 {
namespace {

constexpr int kThreads = 256, kHeads = 2;

struct RopeArgs {
    const void* x;
    int64_t x_batch, x_tok, x_head;      // steps in elements
    const float2* cis;                   // [rows, R / 2]
    int64_t rows;
    const long long* pos;                // of token t of batch b at pos[b * pos_batch + t * pos_tok], or null: t
    int64_t pos_batch, pos_tok;
    void* out;                           // [B, T, H, D]
    int N, H, D, R;                      // N = B * T
    int slices, units, tokens;           // of heads, of a head, of a block
    int half_layout, conj;
    FastDiv per_unit, per_token, per_batch;
};

template <typename T, int P, bool HALF>
__global__ void __launch_bounds__(kThreads, 4) rope_kernel(const RopeArgs a) {
    after_predecessor();
    // item = (token, slice of heads, unit)
    const unsigned token0 = blockIdx.x * (unsigned)a.tokens, tokens = min((unsigned)a.tokens, (unsigned)a.N - token0);
    for (unsigned i = threadIdx.x; i < tokens * a.per_token.d; i += kThreads) {
        const unsigned in = a.per_token.div(i), item = i - in * a.per_token.d, token = token0 + in;
        const int slice = (int)a.per_unit.div(item), u = (int)item - slice * a.units;
        const unsigned b = a.per_batch.div(token), t = token - b * a.per_batch.d;
        const long long p = a.pos ? a.pos[b * a.pos_batch + t * a.pos_tok] : (long long)t;
        int off_a, off_b;
        piece_offsets<P>(u, a.R, a.D, off_a, off_b);
        const T* const src = static_cast<const T*>(a.x) + b * a.x_batch + t * a.x_tok;
        Piece<T, P> x[kHeads], y[kHeads];
#pragma unroll
        for (int j = 0; j < kHeads; ++j) {
            const int h = slice + j * a.slices;
            if (h < a.H) {
                x[j].load(src + h * a.x_head + off_a);
                y[j].load(src + h * a.x_head + off_b);
            }
        }
        const bool inside = p >= 0 && p < a.rows;             // a position outside the table: zeros
        if (!inside) {
#pragma unroll
            for (int j = 0; j < kHeads; ++j) x[j].clear(), y[j].clear();
        } else if (u < a.R / (2 * P)) {
            Angles<P> g = load_angles<P>(a.cis + p * (a.R / 2), u, a.R, HALF);
            if (a.conj) {
#pragma unroll
                for (int e = 0; e < P; ++e) g.s[e] = -g.s[e];
            }
#pragma unroll
            for (int j = 0; j < kHeads; ++j) turn_pieces<T, P>(x[j], y[j], g, HALF);
        }
        T* const dst = static_cast<T*>(a.out) + (int64_t)token * a.H * a.D;
#pragma unroll
        for (int j = 0; j < kHeads; ++j) {
            const int h = slice + j * a.slices;
            if (h < a.H) {
                x[j].store(dst + (int64_t)h * a.D + off_a);
                y[j].store(dst + (int64_t)h * a.D + off_b);
            }
        }
    }
}

// Any even R and any D, of any alignment: one feature a thread.
template <typename T>
__device__ __forceinline__ float to_float(T v) { return static_cast<float>(v); }
template <typename T>
__global__ void __launch_bounds__(kThreads) rope_single_kernel(const RopeArgs a) {
    after_predecessor();
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x, per_token = (int64_t)a.H * a.D;
    const int64_t token = i / per_token;
    if (token >= a.N) return;
    const int hd = (int)(i - token * per_token), h = hd / a.D, d = hd - h * a.D;
    const unsigned b = a.per_batch.div((unsigned)token), t = (unsigned)token - b * a.per_batch.d;
    const long long p = a.pos ? a.pos[b * a.pos_batch + t * a.pos_tok] : (long long)t;
    T* const dst = static_cast<T*>(a.out) + i;
    if (p < 0 || p >= a.rows) {
        *dst = static_cast<T>(0.0f);
        return;
    }
    const T* const src = static_cast<const T*>(a.x) + b * a.x_batch + t * a.x_tok + h * a.x_head;
    if (d >= a.R) {
        *dst = src[d];
        return;
    }
    const int half = a.R / 2, pair = a.half_layout ? (d < half ? d : d - half) : d / 2;
    const bool second = a.half_layout ? d >= half : (d & 1) != 0;
    const int first = a.half_layout ? pair : 2 * pair, other = a.half_layout ? pair + half : first + 1;
    const float2 cs = __ldg(a.cis + p * half + pair);
    float x = to_float(src[first]), y = to_float(src[other]);
    turn(x, y, cs.x, a.conj ? -cs.y : cs.y);
    *dst = static_cast<T>(second ? y : x);
}

template <typename T, int P>
int launch(RopeArgs a, cudaStream_t st) {
    a.units = a.D / (2 * P);
    a.slices = (a.H + kHeads - 1) / kHeads;
    const int64_t per_token = (int64_t)a.slices * a.units;
    a.tokens = (int)(per_token >= kThreads ? 1 : kThreads / per_token);
    a.per_unit = FastDiv(a.units);
    a.per_token = FastDiv(per_token);
    const unsigned grid = (unsigned)(((int64_t)a.N + a.tokens - 1) / a.tokens);
    return a.half_layout ? launch_chained(rope_kernel<T, P, true>, grid, kThreads, 0, st, a) : launch_chained(rope_kernel<T, P, false>, grid, kThreads, 0, st, a);
}

template <typename T>
int launch_type(const RopeArgs& a, cudaStream_t st) {
    // pieces of 8, 4 or 2 features: the widest that divides both parts of a head and begins on its boundaries everywhere
    auto fits = [&](int P) {
        const size_t bytes = sizeof(T) * P > 16 ? 16 : sizeof(T) * P;
        const int64_t steps[3] = {a.x_batch, a.x_tok, a.x_head};
        bool ok = a.R % (2 * P) == 0 && a.D % (2 * P) == 0 && aligned(a.x, bytes) && aligned(a.out, bytes);
        for (int64_t s : steps) ok = ok && s * (int64_t)sizeof(T) % (int64_t)bytes == 0;
        return ok && (int64_t)((a.H + kHeads - 1) / kHeads) * (a.D / (2 * P)) < (1 << 30);
    };
    if constexpr (sizeof(T) == 2)
        if (fits(8)) return launch<T, 8>(a, st);
    if (fits(4)) return launch<T, 4>(a, st);
    if (fits(2)) return launch<T, 2>(a, st);
    const int64_t blocks = ((int64_t)a.N * a.H * a.D + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffff) return fail(BI8_ERR_LIMIT, "rope: %d tokens exceed one launch", a.N);
    return launch_chained(rope_single_kernel<T>, (unsigned)blocks, kThreads, 0, st, a);
}

}  // namespace

int launch_rope(const void* x, int dt, int64_t x_batch, int64_t x_tok, int64_t x_head, const float* cis, int64_t rows, int64_t R, const long long* pos,
                int64_t pos_batch, int64_t pos_tok, void* out, int64_t B, int64_t T, int64_t H, int64_t D, int half_layout, int conj, cudaStream_t st) {
    RopeArgs a{};
    a.x = x;
    a.x_batch = x_batch;
    a.x_tok = x_tok;
    a.x_head = x_head;
    a.cis = reinterpret_cast<const float2*>(cis);
    a.rows = rows;
    a.pos = pos;
    a.pos_batch = pos_batch;
    a.pos_tok = pos_tok;
    a.out = out;
    a.H = (int)H;
    a.D = (int)D;
    a.R = (int)R;
    a.half_layout = half_layout;
    a.conj = conj;
    if (B * T > 0x7fffffff) return fail(BI8_ERR_LIMIT, "rope: %lld tokens exceed one launch", (long long)(B * T));
    a.N = (int)(B * T);
    a.per_batch = FastDiv(T);
    if (dt == BI8_F32) return launch_type<float>(a, st);
    return dt == BI8_BF16 ? launch_type<__nv_bfloat16>(a, st) : launch_type<__half>(a, st);
}

}  // namespace bi8
