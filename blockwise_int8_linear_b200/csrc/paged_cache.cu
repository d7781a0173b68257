// Rotary positions of new tokens' q and k (rope.cuh) and the append of k and v to a paged cache, in one launch, for the packed tokens of
// any number of sequences.
//
// Bound by memory: q, k and v read once, q and the cache's rows written once.  A thread has two pieces of eight features in kHeads heads of one token, as in
// the rotation alone.  A block's tokens find their sequences together: its threads read all of cu side by side and each writes down the tokens that its
// sequences have here, one round of loads instead of a search.  4 x 2048 tokens of 32 + 2 x 32 heads of 128: 77 us, 80 % of a copy's bandwidth; 128 single
// tokens: 2.4 us in a graph.
#include "paged_common.cuh"
#include "rope.cuh"

#include <type_traits>

namespace bi8 {
namespace {

constexpr int kThreads = 256, kHeads = 2, kMaxTokens = 64, P = 8;

struct PagedAppendArgs {
    const void* qkv;             // [N, Hq + 2 Hkv, D]
    int64_t x_tok, x_head;
    const float2* cis;
    int64_t cis_rows;
    void* q_out;                 // [N, Hq, D]
    bi8_paged_cache cache;
    Sequences seq;
    int Hq, Hkv, D, R;
    int slices, units, tokens;   // tokens of a block
    FastDiv per_unit, per_token;
};

template <typename T, bool HALF>
__global__ void __launch_bounds__(kThreads, 4) rope_cache_append_paged_kernel(const PagedAppendArgs a) {
    __shared__ int sequence[kMaxTokens];
    after_predecessor();
    const Sequences& s = a.seq;
    const int64_t token_first = (int64_t)blockIdx.x * a.tokens;
    const int token0 = (int)token_first, tokens = (int)min((int64_t)a.tokens, s.N - token_first);
    if (s.cu) {
        if (threadIdx.x < (unsigned)tokens) sequence[threadIdx.x] = s.B;
        __syncthreads();
        for (int b = threadIdx.x; b < s.B; b += kThreads) {
            const int lo = max(s.first_token(b), token0), hi = min(s.first_token(b + 1), token0 + tokens);
            for (int t = lo; t < hi; ++t) sequence[t - token0] = b;
        }
        __syncthreads();
    }
    const int H = a.Hq + 2 * a.Hkv;
    for (unsigned i = threadIdx.x; i < (unsigned)tokens * a.per_token.d; i += kThreads) {
        const unsigned in = a.per_token.div(i), item = i - in * a.per_token.d;
        const int slice = (int)a.per_unit.div(item), u = (int)item - slice * a.units, token = token0 + (int)in;
        const int b = s.cu ? sequence[in] : (int)s.tokens.div((unsigned)token);
        const int first = s.first_token(b), n = s.first_token(b + 1) - first;
        const long long position = s.first_position(b, n) + (token - first);
        // positions that the angles, the sequence's table or the cache do not have: nothing is written, the query is zero
        bool inside = b < s.B && position >= 0 && position < s.max_len && position < a.cis_rows;
        const int row = inside ? (int)position : 0, in_table = (int)s.page.div((unsigned)row), in_page = row - in_table * (int)s.page.d;
        const int page = inside ? s.pages[b * s.pages_step + in_table] : 0;
        inside = inside && page >= 0 && page < a.cache.pages;

        int off_a, off_b;
        piece_offsets<P>(u, a.R, a.D, off_a, off_b);
        const T* const src = static_cast<const T*>(a.qkv) + token * a.x_tok;
        Piece<T, P> x[kHeads], y[kHeads];
#pragma unroll
        for (int j = 0; j < kHeads; ++j) {
            const int h = slice + j * a.slices;
            if (h < H) {
                x[j].load(src + h * a.x_head + off_a);
                y[j].load(src + h * a.x_head + off_b);
            }
        }
        if (!inside) {
#pragma unroll
            for (int j = 0; j < kHeads; ++j) x[j].clear(), y[j].clear();
        } else if (u < a.R / (2 * P)) {
            const Angles<P> g = load_angles<P>(a.cis + position * (a.R / 2), u, a.R, HALF);
#pragma unroll
            for (int j = 0; j < kHeads; ++j)
                if (slice + j * a.slices < a.Hq + a.Hkv) turn_pieces<T, P>(x[j], y[j], g, HALF);
        }
        const bi8_paged_cache& c = a.cache;
#pragma unroll
        for (int j = 0; j < kHeads; ++j) {
            const int h = slice + j * a.slices;
            T* dst;
            if (h < a.Hq) {
                dst = static_cast<T*>(a.q_out) + ((int64_t)token * a.Hq + h) * a.D;
            } else if (h < H && inside) {
                const int kh = h - a.Hq;
                dst = kh < a.Hkv ? static_cast<T*>(c.k) + page * c.k_page + kh * c.k_head + in_page * c.k_row
                                 : static_cast<T*>(c.v) + page * c.v_page + (kh - a.Hkv) * c.v_head + in_page * c.v_row;
            } else {
                continue;
            }
            x[j].store(dst + off_a);
            y[j].store(dst + off_b);
        }
    }
}

}  // namespace

int launch_rope_cache_append_paged(const void* qkv, int dt, int64_t x_tok, int64_t x_head, const float* cis, int64_t cis_rows, int64_t R, int half_layout,
                                   void* q_out, const bi8_paged_cache* cache, const Sequences& seq, int64_t Hq, int64_t D, cudaStream_t st) {
    PagedAppendArgs a{};
    a.qkv = qkv;
    a.x_tok = x_tok;
    a.x_head = x_head;
    a.cis = reinterpret_cast<const float2*>(cis);
    a.cis_rows = cis_rows;
    a.q_out = q_out;
    a.cache = *cache;
    a.seq = seq;
    a.Hq = (int)Hq;
    a.Hkv = (int)cache->heads;
    a.D = (int)D;
    a.R = (int)R;
    a.units = (int)D / (2 * P);
    a.slices = (int)((Hq + 2 * cache->heads + kHeads - 1) / kHeads);
    const int64_t per_token = (int64_t)a.slices * a.units;
    a.tokens = (int)(per_token >= kThreads ? 1 : kThreads / per_token);
    if (a.tokens > kMaxTokens) a.tokens = kMaxTokens;
    a.per_unit = FastDiv(a.units);
    a.per_token = FastDiv(per_token);
    const unsigned grid = (unsigned)(((int64_t)seq.N + a.tokens - 1) / a.tokens);
    auto go = [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        return half_layout ? launch_chained(rope_cache_append_paged_kernel<T, true>, grid, kThreads, 0, st, a)
                           : launch_chained(rope_cache_append_paged_kernel<T, false>, grid, kThreads, 0, st, a);
    };
    return dt == BI8_BF16 ? go(static_cast<__nv_bfloat16*>(nullptr)) : go(static_cast<__half*>(nullptr));
}

}  // namespace bi8
