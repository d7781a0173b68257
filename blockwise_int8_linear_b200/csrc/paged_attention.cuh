// What both attention kernels over a paged cache take (paged_attention.cu for a few queries of a cache head, paged_attention_tc.cu for many).
#pragma once

#include "paged_common.cuh"

namespace bi8 {

struct PagedAttnArgs {
    const void* q;               // [N, Hq, D]
    int64_t q_tok, q_head;       // steps in elements
    bi8_paged_cache cache;
    Sequences seq;
    void* out;                   // [N, Hq, D]
    Partials part;
    int Hq, Hkv, G;
    int shares, tiles;
    bool by_length;              // both kernels run, each for its sequences: those of at most kFewQueries queries a cache head, and the others
    bool mark;                   // the kernel for few queries tells the join that its results are in place
    float scale_log2;            // |scale| * log2(e), not 0
    uint32_t q_keep, q_flip;     // of two packed queries: bits to keep (none where the scale is 0) and signs to change
    FastDiv group, heads, per_share, per_sequence, sequences;
};

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// The number of rows that query t of a sequence sees, counted from the cache's first, by the position of the sequence's first new token.  (Tokens that belong to
// nobody have positions below 0.)
__device__ __forceinline__ int rows_seen(const Sequences& s, long long first_position, int t) {
    const long long r = first_position + t + 1;
    return (int)(r < 0 ? 0 : r > s.max_len ? s.max_len : r);
}

// The kernel for many queries gives a tile one share for as many rows of the cache: two of its steps, four with heads of 256 features.
constexpr int kShareRows = 256;
int paged_many_tile(int64_t D);          // queries of one of its CTAs
constexpr int kFewQueries = 16;

// Rows of the newest tokens are seen by some queries of a tile and not by others, and in a matrix product a weight of 0 times an infinity is none.  So
// values that are not finite are taken out of those rows before the product (the row is noted, counted from the first that not all
// queries see) and given to the queries that see them when the sums are done: what an infinite value times a positive weight adds is itself.
template <typename T, bool L2>
__device__ __forceinline__ float not_finite(const PagedAttnArgs& a, const int* pages, int row, int h, int d) {      // that value, 0 for a finite one
    const int in_table = (int)a.seq.page.div((unsigned)row), page = load<L2>(pages + in_table);
    if (page < 0 || page >= a.cache.pages) return 0.0f;
    const unsigned short* const v =
        static_cast<const unsigned short*>(a.cache.v) + page * a.cache.v_page + h * a.cache.v_head + (int64_t)(row - in_table * (int)a.seq.page.d) * a.cache.v_row;
    const unsigned short x = load<L2>(v + d);
    return (x & 0x7fffu) >= F16Bits<T>::kInf ? F16Bits<T>::one(x) : 0.0f;
}

int launch_paged_few(const PagedAttnArgs& a, int dt, int64_t D, cudaStream_t st);
int launch_paged_many(const PagedAttnArgs& a, int dt, int64_t D, cudaStream_t st);

}  // namespace bi8
