// Attention over the paged 8-bit cache for any head size up to 256, any strides and alignment
// (b200_kv_attention_generic_launch): one warp per row and query head, one key at a time, the softmax's
// running maximum and sum and the weighted values in f32 registers.
#include "kv_cache.cuh"
#include "launch.hpp"

namespace b200 {
namespace {

constexpr int PER_LANE = 8; // 256 / 32

__global__ void __launch_bounds__(128) kv_attention_generic_kernel(const __grid_constant__ b200_kv_attention_params_t p) {
    const b200_kv_cache_t &c = p.cache;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, qh = blockIdx.y, dim = (int)c.dim;
    if (row >= p.rows) return;
    int b = -1;
    for (int base = 0; base < c.seqs; base += 32) {
        const int i = base + lane;
        const bool in = i < c.seqs && c.offsets[i] <= row && row < c.offsets[i + 1];
        const uint32_t m = __ballot_sync(~0u, in);
        if (m) {
            b = base + __ffs(m) - 1;
            break;
        }
    }
    if (b < 0) return;
    const seq_t s = load_seq(c, b, p.rows);
    const int last = s.first + (int)(row - s.begin); // the newest token that the row sees
    const int head = qh / (int)(p.q_heads / c.heads);
    float q[PER_LANE], o[PER_LANE];
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
        const int e = lane + 32 * i;
        q[i] = e < dim ? load_f32(p.query_dt, p.query, row * p.query_s0 + qh * p.query_s1 + e) : 0.f;
        o[i] = 0.f;
    }
    float top = -INFINITY, sum = 0.f;
    bool bad = false;
    for (int at = 0; at <= last; ++at) {
        int slot;
        const int phys = page_of(c, b, at, slot);
        if (phys < 0) {
            bad = true;
            if (at / (int)c.page >= c.table_cols) break; // nothing further is in the table
            continue;
        }
        const int64_t place = (int64_t)phys * c.s_page + head * c.s_head + (int64_t)slot * c.s_slot;
        const uint8_t *k = (const uint8_t *)c.key + place, *v = (const uint8_t *)c.value + place;
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i)
            if (lane + 32 * i < dim) dot = fmaf(q[i], code_value(c.dt, k[lane + 32 * i]), dot);
#pragma unroll
        for (int w = 16; w; w >>= 1) dot += __shfl_xor_sync(~0u, dot, w);
        const int64_t si = (int64_t)phys * c.heads + head;
        const float score = dot * c.key_scale[si] * p.scale;
        if (score > top) {
            const float f = expf(top - score);
            sum *= f;
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i) o[i] *= f;
            top = score;
        }
        // a score of -inf before any other has no weight; NaN goes through
        const float w = score == -INFINITY ? 0.f : expf(score - top);
        sum += w;
        const float wv = w * c.value_scale[si];
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i)
            if (lane + 32 * i < dim) o[i] = fmaf(wv, code_value(c.dt, v[lane + 32 * i]), o[i]);
    }
    if (bad && lane == 0) flag_bad_page(c);
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
        const int e = lane + 32 * i;
        if (e < dim) store1(p.dst_dt, p.dst, row * p.dst_s0 + qh * p.dst_s1 + e, sum == 0.f ? 0.f : o[i] / sum);
    }
}

} // namespace
} // namespace b200

using namespace b200;

extern "C" B200_API int b200_kv_attention_generic_launch(const b200_kv_attention_params_t *p, b200_stream_t stream) {
    if (!p || !kv_cache_ok(p->cache) || p->rows < 0 || p->rows > 0x7fffffff) return B200_ERR_BAD_ARG;
    for (int dt : {p->query_dt, p->dst_dt})
        if (dt != B200_DT_F32 && dt != B200_DT_BF16 && dt != B200_DT_F16) return B200_ERR_UNSUPPORTED;
    if (p->cache.dim > 256 || p->q_heads < 1 || p->q_heads > 65535) return B200_ERR_UNSUPPORTED;
    if (p->q_heads % p->cache.heads) return B200_ERR_BAD_ARG;
    if (p->rows == 0 || p->cache.seqs == 0) return 0;
    if (!p->query || !p->dst) return B200_ERR_BAD_ARG;
    const dim3 grid((unsigned)((p->rows + 3) / 4), (unsigned)p->q_heads);
    kv_attention_generic_kernel<<<grid, 128, 0, (cudaStream_t)stream>>>(*p);
    return after_launch();
}
