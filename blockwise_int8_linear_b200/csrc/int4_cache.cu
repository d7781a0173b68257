// Rotary embedding of new tokens' q and k and the append of k and v to a key/value cache held in 4-bit blocks.
//
// A thread takes eight features of one head of one token: four (even, odd) pairs, rotated in fp32 with every product and sum rounded on
// its own and rounded to the activation type, as in the 16-bit cache's append.  A block of 64 is eight neighbouring lanes; k and v
// are quantized from those values (int4_common.cuh) and go to row pos + t of their sequence.  Positions are read from device memory, so
// the launch can be captured and replayed while they advance.
#include "int4_common.cuh"

#include <type_traits>

namespace bi8 {
namespace {

constexpr int kThreads = 256;

struct AppendArgs {
    const void* qkv;             // [B, T, Hq + 2 Hkv, D]
    const float2* cis;           // [cis_rows, D / 2]
    int64_t rows;                // positions that the table and the cache have
    const long long* pos;
    int64_t pos_step;
    void* q_out;                 // [B, Hq, T, D]
    bi8_int4_cache cache;
    unsigned units;
    int T, Hq, Hkv, D;
    FastDiv per_head, heads, tokens;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) rope_cache_append_int4_kernel(const AppendArgs a) {
    after_predecessor();
    const unsigned i = blockIdx.x * kThreads + threadIdx.x;
    const bool live = i < a.units;
    const unsigned unit = live ? i : 0u;
    const unsigned hd = a.per_head.div(unit), p = unit - hd * a.per_head.d;            // p: which eight features
    const unsigned tok = a.heads.div(hd), head = hd - tok * a.heads.d;
    const unsigned b = a.tokens.div(tok), t = tok - b * a.tokens.d;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    const long long position = a.pos[b * a.pos_step] + t;
    // a position outside the table or the cache: its key and value are not written, its query is zero
    const bool inside = position >= 0 && position < a.rows;
    const int row = inside ? (int)position : 0;
    if (live && inside) {
        v = ld_nc_v4(static_cast<const T*>(a.qkv) + (int64_t)unit * 8);
        if (head < (unsigned)(a.Hq + a.Hkv)) {
            const float4* cs = reinterpret_cast<const float4*>(a.cis + (int64_t)row * (a.D / 2) + 4 * p);
            const float4 c01 = cs[0], c23 = cs[1];
            const float c[4] = {c01.x, c01.z, c23.x, c23.z}, s[4] = {c01.y, c01.w, c23.y, c23.w};
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x = F16Bits<T>::lo(w[j]), y = F16Bits<T>::hi(w[j]);
                w[j] = F16Bits<T>::pack(__fsub_rn(__fmul_rn(x, c[j]), __fmul_rn(y, s[j])), __fadd_rn(__fmul_rn(x, s[j]), __fmul_rn(y, c[j])));
            }
            v = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    if (!live) return;                                    // units come in whole blocks, and the lanes of a block take the same way
    if (head < (unsigned)a.Hq) {
        *reinterpret_cast<uint4*>(static_cast<T*>(a.q_out) + (int64_t)((b * a.Hq + head) * a.T + t) * a.D + 8 * p) = v;
        return;
    }
    if (!inside) return;
    uint32_t scale;
    const uint32_t codes = quantize8<T, kCacheBlock / 8>(v, 0xffu << (threadIdx.x & 24u), &scale);
    const bool key = head < (unsigned)(a.Hq + a.Hkv);
    const int h = (int)head - a.Hq - (key ? 0 : a.Hkv);
    const bi8_int4_cache& c = a.cache;
    uint8_t* const q = (key ? c.k : c.v) + (int)b * (key ? c.k_batch : c.v_batch) + h * (key ? c.k_head : c.v_head);
    *reinterpret_cast<uint32_t*>(q + (int64_t)row * (a.D / 2) + 4 * p) = codes;
    if ((p & 7u) == 0u) {
        unsigned short* const s = static_cast<unsigned short*>(key ? c.k_state : c.v_state) + (int)b * (key ? c.ks_batch : c.vs_batch) + h * (key ? c.ks_head : c.vs_head);
        s[(int64_t)row * (a.D / kCacheBlock) + (p >> 3)] = (unsigned short)scale;
    }
}

}  // namespace

int launch_rope_cache_append_int4(const void* qkv, int dt, const float* cis, int64_t cis_rows, const long long* pos, int64_t pos_step, void* q_out,
                                  const bi8_int4_cache* cache, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, cudaStream_t st) {
    const int64_t units = B * T * (Hq + 2 * Hkv) * (D / 8);
    if (units > 0x7fffffff - kThreads) return fail(BI8_ERR_LIMIT, "rope_cache_append_int4: %lld values exceed one launch", (long long)units * 8);
    AppendArgs a{};
    a.qkv = qkv;
    a.cis = reinterpret_cast<const float2*>(cis);
    a.rows = cis_rows < cache->max_len ? cis_rows : cache->max_len;
    a.pos = pos;
    a.pos_step = pos_step;
    a.q_out = q_out;
    a.cache = *cache;
    a.units = (unsigned)units;
    a.T = (int)T;
    a.Hq = (int)Hq;
    a.Hkv = (int)Hkv;
    a.D = (int)D;
    a.per_head = FastDiv(D / 8);
    a.heads = FastDiv(Hq + 2 * Hkv);
    a.tokens = FastDiv(T);
    const unsigned grid = (unsigned)((units + kThreads - 1) / kThreads);
    return dt == BI8_BF16 ? launch_chained(rope_cache_append_int4_kernel<__nv_bfloat16>, grid, kThreads, 0, st, a)
                          : launch_chained(rope_cache_append_int4_kernel<__half>, grid, kThreads, 0, st, a);
}

}  // namespace bi8
