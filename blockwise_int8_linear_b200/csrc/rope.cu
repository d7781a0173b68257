// Rotary positions of any tensor [B, T, H, D]: the first R features of every head are turned by the angles of the token's position
// (rope.cuh), the others copied.  The gradient is the same operation with the angles' signs changed (`conj`): the rotation's transpose.
//
// Bound by memory: x read once, the result written once, the table's rows from the caches.  A thread has its two pieces in up to kHeads heads
// of one token, so that a row of the table is read once for those, and as many loads are under way before the first is used.
#include "rope.cuh"

#include <type_traits>

namespace bi8 {
namespace {

constexpr int kThreads = 256, kHeads = 4;

struct RopeArgs {
    const void* x;
    int64_t x_batch, x_tok, x_head;      // steps in elements
    const float2* cis;                   // [rows, R / 2]
    int64_t rows;
    const long long* pos;                // of token t of batch b at pos[b * pos_batch + t * pos_tok], or null: t
    int64_t pos_batch, pos_tok;
    void* out;                           // [B, T, H, D]
    int64_t items;                       // B * T * slices * units
    int H, D, R, slices, units;
    int half_layout, conj;
    FastDiv per_unit, per_slice;
    int64_t T;
};

template <typename T, int P>
__global__ void __launch_bounds__(kThreads) rope_kernel(const RopeArgs a) {
    after_predecessor();
    const int64_t tokens_per_block = a.items;                              // tokens that this launch has
    // a block has kThreads items of consecutive tokens: item = (token, slice of heads, unit)
    const int per_token = a.slices * a.units;
    const int64_t block_first = (int64_t)blockIdx.x * kThreads;
    const int64_t token0 = block_first / per_token;
    const unsigned rest = (unsigned)(block_first - token0 * per_token) + threadIdx.x;
    const unsigned tok_in = a.per_slice.div(rest);
    const int64_t token = token0 + tok_in;
    if (token >= tokens_per_block) return;
    const unsigned item = rest - tok_in * a.per_slice.d;
    const int slice = (int)a.per_unit.div(item), u = (int)item - slice * a.units;
    const int64_t b = token / a.T, t = token - b * a.T;
    const long long p = a.pos ? a.pos[b * a.pos_batch + t * a.pos_tok] : t;
    const bool inside = p >= 0 && p < a.rows;

    int off_a, off_b;
    piece_offsets<P>(u, a.R, a.D, off_a, off_b);
    const bool turned = u < a.R / (2 * P);
    const T* const src = static_cast<const T*>(a.x) + b * a.x_batch + t * a.x_tok;
    T* const dst = static_cast<T*>(a.out) + token * a.H * a.D;
    using V = Piece<T, P>;
    V x[kHeads], y[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        const int h = slice + i * a.slices;
        if (h < a.H && inside) {
            x[i] = *reinterpret_cast<const V*>(src + h * a.x_head + off_a);
            y[i] = *reinterpret_cast<const V*>(src + h * a.x_head + off_b);
        } else {
#pragma unroll
            for (int j = 0; j < P; ++j) x[i].v[j] = y[i].v[j] = RopeType<T>::set(0.0f);      // a position outside the table: zeros
        }
    }
    if (turned && inside) {
        Angles<P> g = load_angles<P>(a.cis + p * (a.R / 2), u, a.R, a.half_layout != 0);
        if (a.conj) {
#pragma unroll
            for (int j = 0; j < P; ++j) g.s[j] = -g.s[j];
        }
#pragma unroll
        for (int i = 0; i < kHeads; ++i)
            if (slice + i * a.slices < a.H) turn_pieces<T, P>(x[i], y[i], g, a.half_layout != 0);
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        const int h = slice + i * a.slices;
        if (h < a.H) {
            *reinterpret_cast<V*>(dst + (int64_t)h * a.D + off_a) = x[i];
            *reinterpret_cast<V*>(dst + (int64_t)h * a.D + off_b) = y[i];
        }
    }
}

// Any even R and any D, of any alignment: one feature a thread.
template <typename T>
__global__ void __launch_bounds__(kThreads) rope_single_kernel(const RopeArgs a) {
    after_predecessor();
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x, per_token = (int64_t)a.H * a.D;
    const int64_t token = i / per_token;
    if (token >= a.items) return;
    const int hd = (int)(i - token * per_token), h = hd / a.D, d = hd - h * a.D;
    const int64_t b = token / a.T, t = token - b * a.T;
    const long long p = a.pos ? a.pos[b * a.pos_batch + t * a.pos_tok] : t;
    T* const dst = static_cast<T*>(a.out) + i;
    if (p < 0 || p >= a.rows) {
        *dst = RopeType<T>::set(0.0f);
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
    float x = RopeType<T>::get(src[first]), y = RopeType<T>::get(src[other]);
    turn(x, y, cs.x, a.conj ? -cs.y : cs.y);
    *dst = RopeType<T>::set(second ? y : x);
}

template <typename T, int P>
int launch(RopeArgs a, int64_t tokens, cudaStream_t st) {
    a.units = a.D / (2 * P);
    a.slices = (a.H + kHeads - 1) / kHeads;
    a.items = tokens;
    a.per_unit = FastDiv(a.units);
    a.per_slice = FastDiv((int64_t)a.slices * a.units);
    const int64_t blocks = (tokens * a.slices * a.units + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffff) return fail(BI8_ERR_LIMIT, "rope: %lld tokens exceed one launch", (long long)tokens);
    return launch_chained(rope_kernel<T, P>, (unsigned)blocks, kThreads, 0, st, a);
}

template <typename T>
int launch_type(const RopeArgs& a, int64_t tokens, cudaStream_t st) {
    // pieces of 8, 4 or 2 features: the widest that divides both parts of a head and begins on its boundaries everywhere
    auto fits = [&](int P) {
        const size_t bytes = sizeof(T) * P > 16 ? 16 : sizeof(T) * P;
        const int64_t steps[3] = {a.x_batch, a.x_tok, a.x_head};
        bool ok = a.R % (2 * P) == 0 && a.D % (2 * P) == 0 && aligned(a.x, bytes) && aligned(a.out, bytes);
        for (int64_t s : steps) ok = ok && s * (int64_t)sizeof(T) % (int64_t)bytes == 0;
        return ok && (int64_t)((a.H + kHeads - 1) / kHeads) * (a.D / (2 * P)) < (1 << 30);
    };
    if (fits(8)) return launch<T, 8>(a, tokens, st);
    if (fits(4)) return launch<T, 4>(a, tokens, st);
    if (fits(2)) return launch<T, 2>(a, tokens, st);
    RopeArgs s = a;
    s.items = tokens;
    const int64_t per_block = kThreads, values = tokens * a.H * a.D, blocks = (values + per_block - 1) / per_block;
    if (blocks > 0x7fffffff) return fail(BI8_ERR_LIMIT, "rope: %lld tokens exceed one launch", (long long)tokens);
    return launch_chained(rope_single_kernel<T>, (unsigned)blocks, kThreads, 0, st, s);
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
    a.T = T;
    if (dt == BI8_F32) return launch_type<float>(a, B * T, st);
    return dt == BI8_BF16 ? launch_type<__nv_bfloat16>(a, B * T, st) : launch_type<__half>(a, B * T, st);
}

}  // namespace bi8
