// Attention over the paged 8-bit cache for few query rows per key head: the choice of a shape
// (kv_attention_mma.cuh has the kernel).
#include "kv_attention_mma.cuh"

namespace b200 {
namespace kv_mma {

#define SHAPE(DP, NB) extern template int run<DP, NB>(const b200_kv_attention_params_t &, int, cudaStream_t);
SHAPE(64, 1) SHAPE(64, 2) SHAPE(128, 1) SHAPE(128, 2) SHAPE(256, 1) SHAPE(256, 2)
#undef SHAPE

namespace {

struct choice_t {
    int dp, nb, blocks; // blocks per SM
};

// Query rows per work item: what a sequence brings on average, tokens times the query heads of a key head.  More rows than an
// item holds are further items that read the tokens again, from L2.  Items of 32 rows were tried: they do not fit the
// registers, and 16 sequences with 2 to 7 tokens, 8 query heads on each key head, took 75 us instead of 58.
choice_t choose(const b200_kv_attention_params_t &p) {
    choice_t c;
    c.dp = p.cache.dim <= 64 ? 64 : p.cache.dim <= 128 ? 128 : 256;
    const int64_t rows = (p.rows + p.cache.seqs - 1) / (p.cache.seqs > 0 ? p.cache.seqs : 1) * (p.q_heads / p.cache.heads);
    c.nb = rows <= 8 ? 1 : 2;
    c.blocks = blocks_of(c.dp, c.nb);
    return c;
}

} // namespace
} // namespace kv_mma
} // namespace b200

using namespace b200;
using namespace b200::kv_mma;

// from the sizes alone
extern "C" B200_API size_t b200_kv_attention_mma_scratch_bytes(const b200_kv_attention_params_t *p) {
    if (!p || p->sm_count < 1 || p->cache.heads < 1) return 0;
    const choice_t c = choose(*p);
    const int blocks = c.blocks * p->sm_count;
    return counter_bytes(blocks) + (size_t)blocks * 2 * part_floats(c.dp, c.nb) * 4;
}

extern "C" B200_API int b200_kv_attention_mma_supported(const b200_kv_attention_params_t *p) {
    const b200_kv_cache_t &c = p->cache;
    if (c.dt != B200_DT_S8 && c.dt != B200_DT_F8_E4M3) return 0;
    for (int dt : {p->query_dt, p->dst_dt})
        if (dt != B200_DT_BF16 && dt != B200_DT_F16) return 0;
    if (c.pages < 1 || c.dim < 16 || c.dim > 256 || c.dim % 16) return 0;
    const uintptr_t bytes = (uintptr_t)c.key | (uintptr_t)c.value | (uintptr_t)c.s_page | (uintptr_t)c.s_head | (uintptr_t)c.s_slot
            | (uintptr_t)p->query | (uintptr_t)p->dst | (uintptr_t)((p->query_s0 | p->query_s1 | p->dst_s0 | p->dst_s1) * 2);
    return bytes % 16 == 0;
}

extern "C" B200_API int b200_kv_attention_mma_launch(const b200_kv_attention_params_t *p, b200_stream_t stream) {
    if (!p || !kv_cache_ok(p->cache) || p->rows < 0 || p->rows > 0x7fffffff) return B200_ERR_BAD_ARG;
    if (!b200_kv_attention_mma_supported(p)) return B200_ERR_UNSUPPORTED;
    if (p->q_heads < 1 || p->q_heads % p->cache.heads || p->sm_count < 1) return B200_ERR_BAD_ARG;
    if (p->rows * (p->q_heads / p->cache.heads) > 0x7fffff00) return B200_ERR_TOO_LARGE;
    if (p->rows == 0 || p->cache.seqs == 0) return 0;
    if (!p->query || !p->dst || !p->scratch || p->scratch_bytes < b200_kv_attention_mma_scratch_bytes(p)) return B200_ERR_BAD_ARG;
    const choice_t c = choose(*p);
    const int blocks = c.blocks * p->sm_count;
    cudaStream_t cs = (cudaStream_t)stream;
    if (!p->scratch_zeroed) {
        const cudaError_t e = cudaMemsetAsync(p->scratch, 0, counter_bytes(blocks), cs);
        if (e != cudaSuccess) return (int)e;
    }
    switch (c.dp * 8 + c.nb) {
        case 64 * 8 + 1: return run<64, 1>(*p, blocks, cs);
        case 64 * 8 + 2: return run<64, 2>(*p, blocks, cs);
        case 128 * 8 + 1: return run<128, 1>(*p, blocks, cs);
        case 128 * 8 + 2: return run<128, 2>(*p, blocks, cs);
        case 256 * 8 + 1: return run<256, 1>(*p, blocks, cs);
        default: return run<256, 2>(*p, blocks, cs);
    }
}
