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
    int64_t cis_rows;
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
    const long long row = a.pos[b * a.pos_step] + t;
    // a position outside the table or the cache: its key and value are not written, its query is zero
    const bool inside = row >= 0 && row < a.cache.max_len && row < a.cis_rows;
    if (live && inside) {
        v = ld_nc_v4(static_cast<const T*>(a.qkv) + (int64_t)unit * 8);
        if (head < (unsigned)(a.Hq + a.Hkv)) {
            const float4* cs = reinterpret_cast<const float4*>(a.cis + row * (a.D / 2) + 4 * p);
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
    uint32_t scale;
    const uint32_t codes = quantize8<T>(v, kCacheBlock / 8, &scale);     // every lane takes part
    if (!live) return;
    if (head < (unsigned)a.Hq) {
        *reinterpret_cast<uint4*>(static_cast<T*>(a.q_out) + (((int64_t)b * a.Hq + head) * a.T + t) * a.D + 8 * p) = v;
        return;
    }
    if (!inside) return;
    const bool key = head < (unsigned)(a.Hq + a.Hkv);
    const int64_t h = head - a.Hq - (key ? 0 : a.Hkv);
    const bi8_int4_cache& c = a.cache;
    uint8_t* q = key ? c.k + b * c.k_batch + h * c.k_head : c.v + b * c.v_batch + h * c.v_head;
    unsigned short* s = key ? static_cast<unsigned short*>(c.k_state) + b * c.ks_batch + h * c.ks_head
                            : static_cast<unsigned short*>(c.v_state) + b * c.vs_batch + h * c.vs_head;
    *reinterpret_cast<uint32_t*>(q + row * (a.D / 2) + 4 * p) = codes;
    if ((p & 7u) == 0u) s[row * (a.D / kCacheBlock) + (p >> 3)] = (unsigned short)scale;
}

}  // namespace

int launch_rope_cache_append_int4(const void* qkv, int dt, const float* cis, int64_t cis_rows, const long long* pos, int64_t pos_step, void* q_out,
                                  const bi8_int4_cache* cache, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, cudaStream_t st) {
    const int64_t units = B * T * (Hq + 2 * Hkv) * (D / 8);
    if (units > 0x7fffffff - kThreads) return fail(BI8_ERR_LIMIT, "rope_cache_append_int4: %lld values exceed one launch", (long long)units * 8);
    AppendArgs a{};
    a.qkv = qkv;
    a.cis = reinterpret_cast<const float2*>(cis);
    a.cis_rows = cis_rows;
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
