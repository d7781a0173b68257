// What the kernels of the paged key/value cache share: which sequence a token or a tile of queries belongs to, and where a row lies.
//
// New tokens of all sequences lie one behind the other: those of sequence b are cu[b] to cu[b + 1], or T each.  A sequence has lengths[b]
// rows, the last of which are its new tokens' own.  What the device's numbers say is never trusted further than the tensors reach: tokens
// are clamped to N, lengths to the table's width, and page numbers that are no page's write nothing and read as zeros.
#pragma once

#include "int4_common.cuh"

namespace bi8 {

// Loads from the L2, past the SM's own cache: for a kernel that begins without a wait of its own (bi8_common.cuh).
__device__ __forceinline__ long long ld_l2(const long long* p) {
    long long v;
    asm volatile("ld.relaxed.gpu.global.s64 %0, [%1];" : "=l"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ int ld_l2(const int* p) {
    int v;
    asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ unsigned short ld_l2(const unsigned short* p) {
    unsigned short v;
    asm volatile("ld.relaxed.gpu.global.u16 %0, [%1];" : "=h"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint4 ld_l2(const uint4* p) {
    uint4 v;
    asm volatile("ld.relaxed.gpu.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
template <bool L2, typename V>
__device__ __forceinline__ V load(const V* p) {
    if constexpr (L2) return ld_l2(p);
    else return *p;
}

struct Sequences {
    const long long* lengths;
    const long long* cu;         // B + 1 first tokens, or null: T tokens each
    const long long* starts;     // or null: 0
    const int* pages;            // [B, width], rows pages_step apart
    int64_t lengths_step, starts_step, pages_step;
    int B, N, T;
    int max_len;                 // rows that a table row has room for
    FastDiv page, tokens;        // rows of a page; tokens of a sequence without cu

    // cu[0] is 0 whatever it says; tokens behind the last sequence's belong to sequence B, which has no rows
    template <bool L2 = false>
    __device__ __forceinline__ int first_token(int b) const {
        if (b <= 0) return 0;
        if (b > B) return N;
        if (!cu) return b * T;
        const long long v = load<L2>(cu + b);
        return (int)(v < 0 ? 0 : v > N ? N : v);
    }
    // position of a sequence's first new token; any number
    template <bool L2 = false>
    __device__ __forceinline__ long long first_position(int b, int n) const { return b < B ? load<L2>(lengths + b * lengths_step) - n : -n; }
    template <bool L2 = false>
    __device__ __forceinline__ int start(int b) const {
        if (!starts || b >= B) return 0;
        const long long v = load<L2>(starts + b * starts_step);
        return (int)(v < 0 ? 0 : v > max_len ? max_len : v);
    }
};

// Tiles of up to `rows` queries each (G of a cache head for every token) of one sequence.  With cu the tiles of sequence b are numbered from
// floor(cu[b] G / rows) + b, which leaves room for every sequence's last tile, and some numbers unused.
struct QueryTile {
    int b, n, token0;            // sequence, its tokens, the first of them
    int row0, rows;              // the tile's queries among the sequence's n * G; rows 0: nothing to do
};

// Called by whole warps.
__device__ __forceinline__ QueryTile find_tile(const Sequences& s, int tile, int G, int rows, const FastDiv& per_sequence) {
    QueryTile t;
    if (!s.cu) {
        t.b = (int)per_sequence.div((unsigned)tile);
        t.row0 = (tile - t.b * (int)per_sequence.d) * rows;
    } else {
        // the last sequence whose tiles begin at or before this number, 32 sequences at a time
        auto begin = [&](int b) { return (int)((long long)s.first_token(b) * G / rows) + b; };
        int lo = 0, hi = s.B + 1;
        while (hi - lo > 1) {
            const int step = (hi - lo + 31) >> 5, at = lo + (int)(threadIdx.x & 31u) * step;
            const unsigned before = __ballot_sync(0xffffffffu, at < hi && begin(at) <= tile);
            const int n = max(__popc(before), 1);
            lo += (n - 1) * step;
            hi = min(hi, lo + step);
        }
        t.b = lo;
        t.row0 = (tile - begin(lo)) * rows;
    }
    t.token0 = s.first_token(t.b);
    t.n = max(s.first_token(t.b + 1) - t.token0, 0);
    const long long left = (long long)t.n * G - t.row0;
    t.rows = (int)(left < 0 || t.row0 < 0 ? 0 : left > rows ? rows : left);
    return t;
}

inline int64_t tile_count(int64_t B, int64_t N, int64_t G, int64_t rows, bool packed) {
    return packed ? N * G / rows + B + 1 : B * ((N / B * G + rows - 1) / rows);
}

// Where attention's kernels put what several shares of a sequence's rows have to be joined from.  The sums of query `row` (token * Hq + head)
// in share k are at ((k * N * Hq) + row) * D, its maximum (in powers of two) and total at the same place among the pairs behind them.
struct Partials {
    float* sums;
    float2* stats;
    int64_t rows;                // N * Hq
};
constexpr float kWritten = -1.0f;     // the total of a query whose result is in place already

int launch_paged_join(const Partials& p, int shares, void* out, int dt, int64_t D, cudaStream_t st);

}  // namespace bi8
