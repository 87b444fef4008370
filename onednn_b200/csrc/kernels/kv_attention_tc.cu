// Attention over the paged 8-bit cache for many query rows per key head (b200_kv_attention_tc_launch): prompts.
// Bound by the tensor cores and, next to them, by the exponentials.
//
// A work item (kv_line.cuh) has 256 query rows, tokens x the query heads of a key head, in two tiles of 128, so that a
// tile of keys and values is converted once for 256 rows.  Per 128 tokens and tile t, on tcgen05.mma (f16 in,
// f32 accumulators in tensor memory):
//   S_t = Q_t K^T        128 x 128 x dim, both operands in shared memory, K-major
//   O_t += P_t V         128 x dim x 128, P from tensor memory (over S, where it was computed), V as it lies, N-major
//
//   warps 0-3, 4-7   softmax of tile 0, 1: one thread per row, so maximum and sum need no exchange; queries
//                    on the way in, results on the way out
//   warps 8-11       codes from the pages to f16 tiles in shared memory (exact), a tile ahead in registers
//   warp 12          one thread issues all MMAs: QK_0(j+1) behind PV_0(j), QK_1(j+1) behind PV_1(j), so that one
//                    tile's softmax runs beside the other's products
//
// The two scales stay out of the products.  A page holds a multiple of 16 tokens here, so 16 neighbouring tokens share
// theirs: x = s * (key scale * softmax scale), and the value scale enters the exponent,
// P = 2^(x - m + log2(value scale) - ref), so neither costs an operation per element; the sum takes P back by a
// factor per 16 tokens.  P is f16 relative to 2^8 (m follows the maximum only when that has grown by more, which saves
// most rescaling of O) and to `ref`, a power of two above all value scales.  FINE (f16 results): what P's rounding left
// is multiplied too.
//
// Every wait is bounded; one that runs out sets a bit in the stream's status word and all roles leave.
#include "kv_line.cuh"
#include "launch.hpp"

namespace b200 {
namespace {

using namespace kv_line;

constexpr int TILE = 128, ROWS = 2 * TILE; // query rows of a tile and of an item
constexpr int SOFTMAX_WARPS = 8, CONVERT_WARPS = 4, WARPS = SOFTMAX_WARPS + CONVERT_WARPS + 1, THREADS = WARPS * 32;
constexpr int STAGES = 2;  // of keys and of values
constexpr int CHUNKS = UNIT / 16;
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t WAIT_TRIES = 1u << 19; // of up to 2 us each, suspended in hardware
enum : uint32_t { ST_WAIT = 0x00100000 };

template <int DP>
struct smem_t {
    static constexpr int MAT = UNIT * DP * 2; // a tile of queries, keys or values in f16
    static constexpr int BYTES = (2 + 2 * STAGES) * MAT;
};

// scales of the tokens of a tile, 16 at a time; four tiles deep: the converters are at most two ahead of the slower softmax
struct scales_t {
    float key[CHUNKS];      // below zero: no such page
    float value_log[CHUNKS]; // log2
    float value_inv[CHUNKS];
};

struct ctrl_t {
    uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
    uint64_t k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES];
    uint32_t tmem_base;
    volatile uint32_t abort;
    uint32_t last_part;
    scales_t scales[4];
    int64_t line_words[34];
};

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t *bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity), "r"(2000u)
            : "memory");
    return ok != 0;
}
// false when the wait ran out or another role gave up; the same for all lanes that wait together
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, uint32_t parity, ctrl_t *c, uint32_t *status) {
    for (uint32_t i = 0; i < WAIT_TRIES; ++i) {
        if (mbar_try(bar, parity)) return true;
        if (c->abort) return false;
    }
    c->abort = 1;
    if (status) atomicOr(status, (uint32_t)ST_WAIT);
    return false;
}
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, ctrl_t *c, uint32_t *status) {
    return __all_sync(~0u, mbar_wait(bar, parity, c, status));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
            : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
            : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[32]) {
    asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
            "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
            : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
            "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]),
            "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]),
            "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
            : "r"(addr)
            : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]),
                 "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]),
                 "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]),
                 "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&v)[32]) {
    asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
            "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]),
            "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
            "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]),
            "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(addr)
            : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *v) {
    asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
            "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]),
            "r"(v[14]), "r"(v[15]), "r"(addr)
            : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptor, 128-byte swizzle: 128-byte rows, eight to an atom, atoms `stride` bytes apart along
// the rows; `lead`: between blocks of 128-byte columns (used where the operand is N-major and wider than 64).
__device__ __forceinline__ uint64_t make_desc(uint32_t saddr, uint32_t lead, uint32_t stride) {
    return (uint64_t)((saddr & 0x3ffff) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | (uint64_t)1 << 46
            | (uint64_t)2 << 61;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float lg2(float x) {
    float r;
    asm("lg2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// four codes -> two f16 pairs, exactly (s8: code + 128 in the low byte of 1024, minus 1152)
template <bool S8>
__device__ __forceinline__ uint2 widen(uint32_t w) {
    uint2 r;
    if (S8) {
        w ^= 0x80808080u;
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r.x) : "r"(__byte_perm(w, 0x64646464u, 0x4140)), "r"(0x64806480u));
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r.y) : "r"(__byte_perm(w, 0x64646464u, 0x4342)), "r"(0x64806480u));
    } else {
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r.x) : "h"((uint16_t)w));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r.y) : "h"((uint16_t)(w >> 16)));
    }
    return r;
}
// f16 tiles: [block of 64 dims][row][128 bytes], 16-byte pieces swizzled by the row
__device__ __forceinline__ uint32_t piece_at(int row, int piece) {
    return (uint32_t)((piece >> 3) * (UNIT * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
}

template <int DP, bool S8, bool FINE>
__global__ void __launch_bounds__(THREADS, 1) kv_attention_tc_kernel(const __grid_constant__ b200_kv_attention_params_t p) {
    using S = smem_t<DP>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ ctrl_t ctrl_mem;
    ctrl_t *ctrl = &ctrl_mem;
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *smem_q = smem, *smem_k = smem + 2 * S::MAT, *smem_v = smem_k + STAGES * S::MAT;
    const b200_kv_cache_t &c = p.cache;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t *status = c.status;

    part_t line;
    if (!begin_part<ROWS>(p, line, ctrl->line_words)) return;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ctrl->q_full[i], SOFTMAX_WARPS / 2);
            mbar_init(&ctrl->p_full[i], SOFTMAX_WARPS / 2);
            mbar_init(&ctrl->s_full[i], 1);
            mbar_init(&ctrl->o_full[i], 1);
        }
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&ctrl->k_full[i], CONVERT_WARPS);
            mbar_init(&ctrl->v_full[i], CONVERT_WARPS);
            mbar_init(&ctrl->k_empty[i], 1);
            mbar_init(&ctrl->v_empty[i], 1);
        }
        ctrl->abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == WARPS - 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctrl->tmem_base)), "r"(TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctrl->tmem_base;
    // columns: S_0 | S_1 | O_0 | O_1
    const int group = line.group;

    if (warp < SOFTMAX_WARPS) {
        // ---------------- softmax: row r of tile t ----------------
        const int t = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tmem_s = tmem + lanes + (uint32_t)(t * UNIT), tmem_o = tmem + lanes + 2 * UNIT + (uint32_t)(t * DP);
        const bool bf16 = p.query_dt == B200_DT_BF16;
        float *parts = (float *)((char *)p.scratch + counter_bytes(gridDim.x));
        constexpr size_t part_size = (size_t)ROWS * (DP + 2);
        uint32_t s_phase = 0, o_phase = 0, tile_i = 0; // tile_i: tiles of tokens since the launch
        int64_t at = line.begin;
        bool ok = true; // once a wait has run out, only the barriers among the softmax warps are kept up
        while (at < line.stop) {
            const place_t q = find_item<ROWS>(p, line, at);
            const seq_t s = line.s;
            const int u0 = (int)(at - q.item_begin), u1 = (int)min((int64_t)q.item.units, line.stop - q.item_begin);
            const int rows = (s.end - s.begin) * group - q.tile * ROWS; // that exist from here on
            const bool active = ok && rows > t * TILE;
            const int idx = q.tile * ROWS + t * TILE + r;
            const bool mine = t * TILE + r < rows;
            const int64_t at_row = s.begin + idx / group, at_head = (int64_t)q.head * group + idx % group;
            float m = -INFINITY, l = 0.f, ref = -200.f;
            if (active) {
                // ---- the row's query: to f16 after a power of two that brings its largest element to [1, 2).
                // A negative softmax scale turns the query round, so that factors of the scores are positive.
                const int limit = mine ? s.first + idx / group : -1;
                const int first_limit = __shfl_sync(~0u, limit, 0); // the smallest of the warp's rows that exist
                float factor;
                {
                    uint4 w[DP / 8];
                    uint32_t top = 0;
                    const char *from = (const char *)p.query + (at_row * p.query_s0 + at_head * p.query_s1) * 2;
#pragma unroll
                    for (int i = 0; i < DP / 8; ++i) w[i] = mine && i * 8 < c.dim ? *(const uint4 *)(from + i * 16) : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < DP / 8; ++i) {
                        const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            const float2 f = bf16 ? bf16x2_to_f32(x[h]) : f16x2_to_f32(x[h]);
                            top = max(top, max(__float_as_uint(fabsf(f.x)), __float_as_uint(fabsf(f.y))));
                        }
                    }
                    const int e = top == 0 ? 127 : min(max((int)(top >> 23), 1), 253);
                    float down = __uint_as_float((uint32_t)(254 - e) << 23);
                    if (p.scale < 0.f) down = -down;
                    factor = fabsf(p.scale) * 1.4426950408889634f * __uint_as_float((uint32_t)e << 23);
                    uint8_t *to = smem_q + t * S::MAT;
#pragma unroll
                    for (int i = 0; i < DP / 8; ++i) {
                        const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
                        uint32_t y[4];
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            const float2 f = bf16 ? bf16x2_to_f32(x[h]) : f16x2_to_f32(x[h]);
                            y[h] = pack_f16x2(f.x * down, f.y * down);
                        }
                        *(uint4 *)(to + piece_at(r, i)) = make_uint4(y[0], y[1], y[2], y[3]);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->q_full[t]);

                for (int j = u0; j < u1; ++j, ++tile_i) {
                    if (!(ok = warp_wait(&ctrl->s_full[t], s_phase, ctrl, status))) break;
                    s_phase ^= 1;
                    tc_fence_after();
                    const scales_t &sc = ctrl->scales[tile_i & 3];
                    const bool masked = j * UNIT + UNIT - 1 > first_limit;
                    const int seen = limit - j * UNIT; // columns 0 .. seen are seen
                    // ---- the largest score, and the largest value scale
                    float top = m, vtop = -300.f;
                    bool gaps = false;
#pragma unroll
                    for (int h = 0; h < UNIT / 32; ++h) {
                        uint32_t v[32];
                        tmem_ld32(tmem_s + h * 32, v);
                        if (masked) {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (h * 32 + i > seen) v[i] = 0xff800000u;
                        }
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const float key = sc.key[h * 2 + k];
                            gaps |= key < 0.f;
                            vtop = fmaxf(vtop, sc.value_log[h * 2 + k]);
                            float x = -INFINITY;
#pragma unroll
                            for (int i = 0; i < 16; ++i) x = fmaxf(x, __uint_as_float(v[k * 16 + i]));
                            if (key >= 0.f) top = fmaxf(top, x * fmaxf(key * factor, 1.17549435e-38f));
                        }
                    }
                    // ---- m and ref follow; O and the sum with them
                    const float ref_now = vtop > ref ? ceilf(vtop) + 1.f : ref;
                    const bool follow = top > m + 8.f; // also from -inf
                    const float m_now = follow ? top : m;
                    float fo = 1.f;
                    if (follow || ref_now != ref) {
                        const float d = follow ? ex2(m - m_now) : 1.f;
                        l *= d;
                        fo = d * ex2(ref - ref_now);
                    }
                    m = m_now;
                    ref = ref_now;
                    if (j > u0 && __any_sync(~0u, fo != 1.f)) {
#pragma unroll
                        for (int h = 0; h < DP / 32; ++h) {
                            uint32_t v[32];
                            tmem_ld32(tmem_o + h * 32, v);
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * fo);
                            tmem_st32(tmem_o + h * 32, v);
                        }
                    }
                    // ---- weights
                    const float base = (m == -INFINITY ? 0.f : m) + ref;
                    const float ref_up = ex2(ref);
#pragma unroll
                    for (int h = 0; h < UNIT / 32; ++h) {
                        uint32_t v[32], pw[16], rest[FINE ? 16 : 1];
                        tmem_ld32(tmem_s + h * 32, v);
                        if (masked) {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (h * 32 + i > seen) v[i] = 0xff800000u;
                        }
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const float key = sc.key[h * 2 + k];
                            const float f = fmaxf(key * factor, 1.17549435e-38f);
                            // scales below 2^-60 of the largest count as that: their values round to nothing, their weights stay in the sum
                            const float vl = fmaxf(sc.value_log[h * 2 + k], ref - 60.f);
                            const float off = gaps && key < 0.f ? -INFINITY : vl - base;
                            const float back = fminf(sc.value_inv[h * 2 + k] * ref_up, 1.152921504606847e18f); // 2^60
                            float sum = 0.f;
#pragma unroll
                            for (int i = 0; i < 16; i += 2) {
                                const float x0 = ex2(fmaf(__uint_as_float(v[k * 16 + i]), f, off));
                                const float x1 = ex2(fmaf(__uint_as_float(v[k * 16 + i + 1]), f, off));
                                sum += x0;
                                sum += x1;
                                const uint32_t hi = pack_f16x2(x0, x1);
                                pw[k * 8 + i / 2] = hi;
                                if (FINE) {
                                    const float2 had = f16x2_to_f32(hi);
                                    rest[FINE ? k * 8 + i / 2 : 0] = pack_f16x2(x0 - had.x, x1 - had.y);
                                }
                            }
                            l = fmaf(sum, back, l);
                        }
                        // over the 32 columns just read
                        tmem_st16(tmem_s + h * 32, pw);
                        if (FINE) tmem_st16(tmem_s + h * 32 + 16, rest);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctrl->p_full[t]);
                }
                if (ok) ok = warp_wait(&ctrl->o_full[t], o_phase, ctrl, status);
                o_phase ^= 1;
                tc_fence_after();
            } else {
                tile_i += (uint32_t)(u1 - u0);
            }

            // ---- the row's result, or its part of it
            const bool whole = u0 == 0 && u1 == q.item.units;
            const float up = ref <= -200.f ? 0.f : ex2(ref);
            if (l != l) m = INFINITY; // a NaN among the scores, which no maximum shows
            char *to = (char *)p.dst + (at_row * p.dst_s0 + at_head * p.dst_s1) * 2;
            float *part = parts + (size_t)(blockIdx.x * 2 + (at == line.begin ? 0 : 1)) * part_size;
            const int pr = t * TILE + r; // row of the item
            auto put = [&](int d, const float (&x)[8], float inv) { // eight dims of the result
                if (d >= c.dim) return;
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = x[i] * inv;
                store8(p.dst_dt, to + d * 2, y);
            };
            if (active && ok) {
                const float inv = l == 0.f ? 0.f : up / l;
#pragma unroll
                for (int h = 0; h < DP / 32; ++h) {
                    uint32_t v[32];
                    tmem_ld32(tmem_o + h * 32, v);
                    if (!mine) continue;
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        float x[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) x[k] = __uint_as_float(v[i + k]);
                        if (whole) {
                            put(h * 32 + i, x, inv);
                        } else { // rows side by side, so that a warp's stores are contiguous
                            float4 *d4 = (float4 *)(part + 2 * ROWS) + (h * 32 + i) / 4 * ROWS + pr;
                            d4[0] = make_float4(x[0] * up, x[1] * up, x[2] * up, x[3] * up);
                            d4[ROWS] = make_float4(x[4] * up, x[5] * up, x[6] * up, x[7] * up);
                        }
                    }
                }
                tc_fence_before(); // O may be written again after the next arrival
                if (!whole && mine) part[pr] = m, part[ROWS + pr] = l;
            }
            if (!whole) {
                // an item in several parts: the last block to finish one puts them together, in the order of the parts
                const int c0 = owner(line, q.item_begin), c1 = owner(line, q.item_begin + q.item.units - 1);
                __threadfence();
                asm volatile("bar.sync 1, %0;" ::"n"(SOFTMAX_WARPS * 32) : "memory");
                if (threadIdx.x == 0) {
                    uint32_t *count = (uint32_t *)p.scratch + c0;
                    const bool is_last = atomicAdd(count, 1u) == (uint32_t)(c1 - c0);
                    if (is_last) *count = 0; // as it was found
                    ctrl->last_part = is_last;
                }
                asm volatile("bar.sync 1, %0;" ::"n"(SOFTMAX_WARPS * 32) : "memory");
                const bool is_last = ctrl->last_part;
                asm volatile("bar.sync 1, %0;" ::"n"(SOFTMAX_WARPS * 32) : "memory"); // read before it is set again
                if (is_last && mine) {
                    __threadfence();
                    auto part_of = [&](int b) { return parts + part_index(line, q.item_begin, c0, b) * part_size; };
                    float mm = -INFINITY, ll = 0.f;
                    for (int b = c0; b <= c1; ++b) mm = fmaxf(mm, __ldcg(part_of(b) + pr));
                    for (int b = c0; b <= c1; ++b) {
                        const float mb = __ldcg(part_of(b) + pr), f = mb == -INFINITY ? 0.f : ex2(mb - mm);
                        if (f != 0.f) ll = fmaf(__ldcg(part_of(b) + ROWS + pr), f, ll);
                    }
                    const float inv = ll == 0.f ? 0.f : 1.f / ll;
#pragma unroll 1
                    for (int d = 0; d < DP; d += 32) {
                        float x[4][8];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int k = 0; k < 8; ++k) x[i][k] = 0.f;
                        for (int b = c0; b <= c1; ++b) {
                            const float mb = __ldcg(part_of(b) + pr), f = mb == -INFINITY ? 0.f : ex2(mb - mm);
                            if (f == 0.f) continue;
                            const float4 *d4 = (const float4 *)(part_of(b) + 2 * ROWS) + d / 4 * ROWS + pr;
                            float4 y[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) y[i] = __ldcg(d4 + i * ROWS);
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                float *z = x[i / 2] + (i & 1) * 4;
                                z[0] = fmaf(y[i].x, f, z[0]), z[1] = fmaf(y[i].y, f, z[1]), z[2] = fmaf(y[i].z, f, z[2]), z[3] = fmaf(y[i].w, f, z[3]);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) put(d + i * 8, x[i], inv);
                    }
                }
            }
            at = q.item_begin + u1;
        }
    } else if (warp < SOFTMAX_WARPS + CONVERT_WARPS) {
        // ---------------- codes to f16 ----------------
        // Warp w has tokens 32 w .. of a tile: two runs of 16, each in one page.  CH lanes share a token (16 codes each), so an
        // access of the warp covers 32 / CH tokens.
        constexpr int CH = DP / 16, PER = 32 / CH, LOADS = 32 / PER;
        const int w = warp - SOFTMAX_WARPS, cc = lane % CH, page = (int)c.page;
        const bool takes = cc * 16 < c.dim;
        uint32_t tile_i = 0;
        int64_t at = line.begin;
        bool ok = true;
        while (at < line.stop && ok) {
            const place_t q = find_item<ROWS>(p, line, at);
            const seq_t s = line.s;
            const int u0 = (int)(at - q.item_begin), u1 = (int)min((int64_t)q.item.units, line.stop - q.item_begin);
            const int end = q.item.tokens;
            if (w == 0 && lane == 0 && u0 == 0 && (int64_t)s.first + (s.end - s.begin) > line.capacity) flag_bad_page(c);
            const int32_t *table = c.table + (int64_t)line.seq * c.table_s0;
            const uint8_t *keys = (const uint8_t *)c.key + q.head * c.s_head + cc * 16, *values = (const uint8_t *)c.value + q.head * c.s_head + cc * 16;
            uint4 kr[LOADS], vr[LOADS];
            float ks[2], vs[2];
            // where the two runs of tile j are; below zero: nowhere
            auto find = [&](int j, int64_t (&place)[2], int (&page_at)[2]) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int tok = j * UNIT + w * 32 + h * 16;
                    place[h] = -1;
                    page_at[h] = 0;
                    if (j < u1 && tok < end) {
                        const int n = tok / page, slot = tok - n * page, phys = table[n];
                        if (phys >= 0 && phys < c.pages) place[h] = (int64_t)phys * c.s_page + (int64_t)slot * c.s_slot, page_at[h] = phys;
                        else flag_bad_page(c);
                    }
                }
            };
            auto load = [&](int j, const uint8_t *from, const int64_t (&place)[2], uint4 (&regs)[LOADS]) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const int tok = i * PER + lane / CH, h = tok >> 4; // of the warp's 32
                    regs[i] = make_uint4(0, 0, 0, 0);
                    const int64_t at_run = h ? place[1] : place[0];
                    if (takes && at_run >= 0 && j * UNIT + w * 32 + tok < end)
                        regs[i] = __ldg((const uint4 *)(from + at_run + (int64_t)(tok & 15) * c.s_slot));
                }
            };
            auto load_scales = [&](const int64_t (&place)[2], const int (&page_at)[2]) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int64_t i = (int64_t)page_at[h] * c.heads + q.head;
                    ks[h] = place[h] >= 0 ? c.key_scale[i] : -1.f;
                    vs[h] = place[h] >= 0 ? c.value_scale[i] : 0.f;
                }
            };
            auto convert = [&](const uint4 (&regs)[LOADS], uint8_t *to) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const int row = w * 32 + i * PER + lane / CH;
                    const uint2 a = widen<S8>(regs[i].x), b = widen<S8>(regs[i].y), d = widen<S8>(regs[i].z), e = widen<S8>(regs[i].w);
                    const uint4 lo = make_uint4(a.x, a.y, b.x, b.y), hi = make_uint4(d.x, d.y, e.x, e.y);
                    // two 16-byte pieces; half of the lanes of a row store theirs the other way round: other banks
                    const int swap = cc >> 2 & 1;
                    *(uint4 *)(to + piece_at(row, cc * 2 + swap)) = swap ? hi : lo;
                    *(uint4 *)(to + piece_at(row, cc * 2 + 1 - swap)) = swap ? lo : hi;
                }
            };
            int64_t place[2];
            int page_at[2];
            find(u0, place, page_at);
            load_scales(place, page_at);
            load(u0, keys, place, kr);
            load(u0, values, place, vr);
            for (int j = u0; j < u1; ++j, ++tile_i) {
                const int st = tile_i % STAGES;
                const uint32_t use = tile_i / STAGES;
                // keys, and both scales: a softmax that sees the scores sees them
                if (use > 0 && !(ok = warp_wait(&ctrl->k_empty[st], (use - 1) & 1, ctrl, status))) break;
                if (lane < 2) {
                    const float v = fmaxf(lane ? vs[1] : vs[0], 7.5231638e-37f); // 2^-120
                    scales_t &sc = ctrl->scales[tile_i & 3];
                    sc.key[w * 2 + lane] = lane ? ks[1] : ks[0];
                    sc.value_log[w * 2 + lane] = lg2(v);
                    sc.value_inv[w * 2 + lane] = 1.f / v;
                }
                convert(kr, smem_k + st * S::MAT);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->k_full[st]);
                find(j + 1, place, page_at);
                load_scales(place, page_at);
                load(j + 1, keys, place, kr);
                if (use > 0 && !(ok = warp_wait(&ctrl->v_empty[st], (use - 1) & 1, ctrl, status))) break;
                convert(vr, smem_v + st * S::MAT);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->v_full[st]);
                load(j + 1, values, place, vr);
            }
            at = q.item_begin + u1;
        }
    } else if (lane == 0) {
        // ---------------- the MMAs ----------------
        constexpr uint32_t IDESC = (1u << 4) | ((uint32_t)(TILE >> 4) << 24);
        constexpr uint32_t IDESC_S = IDESC | ((uint32_t)(UNIT >> 3) << 17);
        constexpr uint32_t IDESC_O = IDESC | (1u << 16) | ((uint32_t)(DP >> 3) << 17); // values are N-major
        uint32_t q_phase[2] = {0, 0}, p_phase[2] = {0, 0}, tile_i = 0;
        int64_t at = line.begin;
        bool ok = true;
        auto scores = [&](int t, int st) { // S_t = Q_t K^T
            const uint32_t a = smem_u32(smem_q + t * S::MAT), b = smem_u32(smem_k + st * S::MAT);
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                const uint32_t o = (uint32_t)((k >> 2) * (UNIT * 128) + (k & 3) * 32);
                mma_ss(tmem + t * UNIT, make_desc(a + o, 16, 1024), make_desc(b + o, 16, 1024), IDESC_S, k != 0);
            }
        };
        auto weigh = [&](int t, int st, bool more) { // O_t += P_t V
            const uint32_t b = smem_u32(smem_v + st * S::MAT);
#pragma unroll
            for (int k = 0; k < UNIT / 16; ++k) {
                const uint64_t desc = make_desc(b + k * 2048, UNIT * 128, 1024);
                const uint32_t a = tmem + t * UNIT + (k >> 1) * 32 + (k & 1) * 8;
                mma_ts(tmem + 2 * UNIT + t * DP, a, desc, IDESC_O, more || k != 0);
                if (FINE) mma_ts(tmem + 2 * UNIT + t * DP, a + 16, desc, IDESC_O, 1);
            }
        };
        while (at < line.stop && ok) {
            const place_t q = find_item<ROWS>(p, line, at);
            const seq_t s = line.s;
            const int u0 = (int)(at - q.item_begin), u1 = (int)min((int64_t)q.item.units, line.stop - q.item_begin);
            const int rows = (s.end - s.begin) * group - q.tile * ROWS;
            const int tiles = rows > TILE ? 2 : 1, n = u1 - u0;
            if (!(ok = mbar_wait(&ctrl->k_full[tile_i % STAGES], (tile_i / STAGES) & 1, ctrl, status))) break;
            for (int t = 0; t < tiles && ok; ++t) {
                if (!(ok = mbar_wait(&ctrl->q_full[t], q_phase[t], ctrl, status))) break;
                q_phase[t] ^= 1;
                tc_fence_after();
                scores(t, tile_i % STAGES);
                tc_commit(&ctrl->s_full[t]);
            }
            if (!ok) break;
            tc_commit(&ctrl->k_empty[tile_i % STAGES]);
            for (int j = 0; j < n && ok; ++j, ++tile_i) {
                const int st = tile_i % STAGES, next = (tile_i + 1) % STAGES;
                if (!(ok = mbar_wait(&ctrl->v_full[st], (tile_i / STAGES) & 1, ctrl, status))) break;
                if (j + 1 < n && !(ok = mbar_wait(&ctrl->k_full[next], ((tile_i + 1) / STAGES) & 1, ctrl, status))) break;
                for (int t = 0; t < tiles; ++t) {
                    if (!(ok = mbar_wait(&ctrl->p_full[t], p_phase[t], ctrl, status))) break;
                    p_phase[t] ^= 1;
                    tc_fence_after();
                    weigh(t, st, j > 0);
                    if (j + 1 < n) {
                        scores(t, next);
                        tc_commit(&ctrl->s_full[t]);
                    } else {
                        tc_commit(&ctrl->o_full[t]);
                    }
                }
                if (!ok) break;
                tc_commit(&ctrl->v_empty[st]);
                if (j + 1 < n) tc_commit(&ctrl->k_empty[next]);
            }
            at = q.item_begin + u1;
        }
    }
    // all roles are through (the MMAs too: every one was waited for by way of o_full, unless a wait ran out)
    __syncthreads();
    if (warp == WARPS - 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

template <int DP, bool S8, bool FINE>
int run(const b200_kv_attention_params_t &p, cudaStream_t cs) {
    auto kernel = kv_attention_tc_kernel<DP, S8, FINE>;
    const int bytes = smem_t<DP>::BYTES + 1024;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return (int)e;
    kernel<<<p.sm_count, THREADS, bytes, cs>>>(p);
    return after_launch();
}
template <int DP, bool S8>
int run(const b200_kv_attention_params_t &p, cudaStream_t cs) {
    return p.dst_dt == B200_DT_F16 ? run<DP, S8, true>(p, cs) : run<DP, S8, false>(p, cs);
}

int padded_dim(const b200_kv_attention_params_t &p) { return p.cache.dim <= 64 ? 64 : 128; }

} // namespace
} // namespace b200

using namespace b200;

extern "C" B200_API size_t b200_kv_attention_tc_scratch_bytes(const b200_kv_attention_params_t *p) {
    if (!p || p->sm_count < 1) return 0;
    return counter_bytes(p->sm_count) + (size_t)p->sm_count * 2 * ROWS * (padded_dim(*p) + 2) * 4;
}

extern "C" B200_API int b200_kv_attention_tc_supported(const b200_kv_attention_params_t *p) {
    // what the other kernel takes, with pages of whole runs of 16 tokens, and more query rows per sequence and key head
    // than its items hold
    if (!b200_kv_attention_mma_supported(p) || p->cache.dim > 128 || p->cache.page % 16) return 0;
    return p->cache.seqs > 0 && p->cache.heads > 0 && p->rows / p->cache.seqs * (p->q_heads / p->cache.heads) > 32;
}

extern "C" B200_API int b200_kv_attention_tc_launch(const b200_kv_attention_params_t *p, b200_stream_t stream) {
    if (!p || !kv_cache_ok(p->cache) || p->rows < 0 || p->rows > 0x7fffffff) return B200_ERR_BAD_ARG;
    if (!b200_kv_attention_tc_supported(p)) return B200_ERR_UNSUPPORTED;
    if (p->q_heads < 1 || p->q_heads % p->cache.heads || p->sm_count < 1) return B200_ERR_BAD_ARG;
    if (p->rows * (p->q_heads / p->cache.heads) > 0x7fffff00) return B200_ERR_TOO_LARGE;
    if (p->rows == 0 || p->cache.seqs == 0) return 0;
    if (!p->query || !p->dst || !p->scratch || p->scratch_bytes < b200_kv_attention_tc_scratch_bytes(p)) return B200_ERR_BAD_ARG;
    cudaStream_t cs = (cudaStream_t)stream;
    if (!p->scratch_zeroed) {
        const cudaError_t e = cudaMemsetAsync(p->scratch, 0, counter_bytes(p->sm_count), cs);
        if (e != cudaSuccess) return (int)e;
    }
    const bool s8 = p->cache.dt == B200_DT_S8;
    if (padded_dim(*p) == 64) return s8 ? run<64, true>(*p, cs) : run<64, false>(*p, cs);
    return s8 ? run<128, true>(*p, cs) : run<128, false>(*p, cs);
}
