// Attention over the paged 8-bit cache for many query rows per key head (b200_kv_attention_tc_launch): prompts.
// Bound by the tensor cores and, next to them, by the exponentials.
//
// A work item (kv_line.cuh) has 256 query rows, tokens x the query heads of a key head, in two tiles of 128, so that a
// tile of keys and values is converted once for 256 rows.  Per step of 64 tokens and tile t, on tcgen05.mma (f16 in,
// f32 accumulators in tensor memory):
//   S_t = Q_t K^T        128 x 64 x dim, both operands in shared memory, K-major
//   O_t += P_t V         128 x dim x 64, P from tensor memory (over S, where it was computed), V as it lies, N-major
// S_t has two places, so that a step's scores are there before the softmax is through with the step before; with one
// place of 128 tokens the softmax waited a third of the time for the products between.
//
//   warps 0-3, 4-7   softmax of tile 0, 1: one thread per row, so maximum and sum need no exchange; queries
//                    on the way in, results on the way out
//   warps 8-11       codes from the pages to f16 tiles in shared memory (exact), a tile ahead in registers
//   warps 12, 13     one thread of each issues the MMAs of tile 0, 1: PV(s), then the scores of step s + 2 into the same
//                    place.  (One thread for both tiles was what everything waited for: an MMA takes it some 70 cycles, a
//                    look at a barrier some 300.)
//   warp 14          finds the block's items ahead of all others and lays them out in shared memory
//
// The two scales stay out of the products.  A page holds a multiple of RUN (16 or 8) tokens here, so as many neighbouring tokens
// share theirs: x = s * (key scale * softmax scale) in the exponent's multiply-add, P = w * (value scale * 2^(13 - k)) with
// w = 2^(x - m), two elements at a time, and the sum is of the w.  m and k are the row's own: m follows the largest
// score that the row has seen when that has grown by more than 2^8, which saves most rescaling of O; k is
// not below x + log2(value scale) - m of any token that the row sees.  So P < 2^13, rounded to f16 relative to what the row
// sees, and no page that it does not see, or gives no weight, takes bits from the others (with the value scale in the
// exponent, relative to the largest of all pages, 3 % faster, a page 2^30 above the others took them to zero in rows that
// did not see it).  FINE (f16 results): what P's rounding left is multiplied too.
//
// Measured on one B200: three sequences with 1450, 1029 and 1710 new tokens on 5750, 4647 and 3543, 32 query heads on 8, dim 128, s8,
// bf16: 342 us, 772 Tflop/s of the pairs that causality leaves; 2.6 us per 128 tokens and 256 rows, where the MMAs
// alone take 1.3.  What is left: a softmax step of 64 columns takes a warp 2000 cycles, two of the three warps on a
// scheduler; items begin and end (8 us each) and cut ones are joined (10 us).  Not kept: 16 softmax warps, two threads per row
// (3.6 us per 128 tokens: the converters lost their turns), 8 converter warps (3.6), one issuing thread (2.9).
//
// Every wait is bounded; one that runs out sets a bit in the stream's status word and all roles leave.
#include "kv_f16.cuh"
#include "kv_line.cuh"
#include "launch.hpp"

namespace b200 {
namespace {

using namespace kv_line;

constexpr int TILE = 128, ROWS = 2 * TILE; // query rows of a tile and of an item
constexpr int SOFTMAX_WARPS = 8, CONVERT_WARPS = 4, MMA_WARP = SOFTMAX_WARPS + CONVERT_WARPS, WARPS = MMA_WARP + 4, THREADS = WARPS * 32;
// registers per thread: what the launch gives every warp, and how the four groups of four warps share it
constexpr int REGS = 128, SOFTMAX_REGS = 176, CONVERT_REGS = 104, MMA_REGS = 56;
static_assert(2 * SOFTMAX_REGS + CONVERT_REGS + MMA_REGS <= 4 * REGS && THREADS * REGS <= 65536, "");
constexpr int EXTRA = 3;   // units that an item's queries, filling and draining, and result take besides (8 of 2.5 us)
constexpr int MIN_PART = 2; // units; 2 sequences x 8 tokens over 2600 took 46, 41, 39, 41 us with 1, 2, 4, 6, three short prompts 33, 33, 35, 45
constexpr int STAGES = 2;  // of keys and of values
constexpr int STEP = 64, STEPS = UNIT / STEP; // tokens of a step; steps of a unit, which the converters work on
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t WAIT_TRIES = 1u << 30; // the clock ends a wait long before
constexpr uint64_t WAIT_NS = 4000000000ull; // a warp without rows waits through the other tile's whole segment, which takes milliseconds at most
enum : uint32_t { ST_WAIT = 0x00100000 };

template <int DP>
struct smem_t {
    static constexpr int MAT = UNIT * DP * 2; // a tile of queries, keys or values in f16
    static constexpr int BYTES = (2 + 2 * STAGES) * MAT;
};

// The scales of a tile's tokens, run by run, as the softmax takes them.  Four tiles deep: the converters are at most
// two ahead of the slower softmax.
struct scales_t {
    // x key scale, y 0 (-inf: no such page), z a whole number above log2(value scale), by one at most, w value scale
    float4 chunk[UNIT / 8];
    float above, below; // whole numbers, not below and not above any log2(value scale)
};
constexpr float P_TOP = 13.f; // P stays below 2^13
// of m: x - m in one multiply-add leaves what rounding took from m, at most 2^2 up to here, for which P has room; a row whose m
// goes beyond becomes NaN
// (rounding x first, an operation more per element, has no such end and took 353 us instead of 341)
constexpr float M_MOST = 67108864.f;
constexpr float ROOM = 8.f;   // what m, and with it k, may lag behind
constexpr float K_MIN = -100.f, K_MAX = 121.f; // of k: where all scales that a row sees are below 2^-100, f16's last bits go unused
constexpr float G_MAX = 1.3292280e36f;         // 2^120, of the factor of a run that a row does not see: 0 * infinity is no weight
constexpr float SMALL = 1.0842022e-19f; // 2^-63

// a stretch of an item's tokens: what one block does of it
struct segment_t {
    int begin, rows;   // of the sequence, in the batch; query rows (x group) that exist from the item's first on, 0: no more segments
    int row0, first;   // the item's first query row in the sequence; token of the sequence's first row
    int head, seq;
    int tokens;        // that the item's last row sees
    int u0, u1;        // units
    int whole;         // all of the item's
    int c0, c1;        // the blocks that share the item
    int over;          // whether the sequence has tokens beyond the table
};
constexpr int SEGMENTS = 4;

struct ctrl_t {
    uint64_t seg_full[SEGMENTS], seg_empty[SEGMENTS];
    segment_t segments[SEGMENTS];
    uint64_t q_full[2], s_full[2][STEPS], p_full[2][STEPS], o_done[2][STEPS], join;
    uint64_t k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES];
    uint64_t drained[2];
    uint32_t tmem_base;
    volatile uint32_t abort;
    uint32_t last_part;
    scales_t scales[4];
    int64_t line_words[LINE_WORDS];
};

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
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
    return ok != 0;
}
__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// false when the wait ran out (by the clock) or another role gave up; the same for all lanes that wait together
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, uint32_t parity, ctrl_t *c, uint32_t *status) {
    if (mbar_try(bar, parity)) return true;
    const uint64_t until = now_ns() + WAIT_NS;
    for (uint32_t i = 0; i < WAIT_TRIES; ++i) {
        if (mbar_try(bar, parity)) return true;
        if (c->abort || ((i & 255) == 255 && now_ns() > until)) break;
    }
    if (!c->abort) {
        c->abort = 1;
        if (status) atomicOr(status, (uint32_t)ST_WAIT);
    }
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
__device__ __forceinline__ void tmem_ld32_issue(uint32_t addr, uint32_t (&v)[32]) {
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
}
// all loads before it have arrived
__device__ __forceinline__ void tmem_ld32_wait(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]),
                 "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]),
                 "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]),
                 "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[32]) {
    tmem_ld32_issue(addr, v);
    tmem_ld32_wait(v);
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *v) {
    asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
            "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]),
            "r"(v[14]), "r"(v[15]), "r"(addr)
            : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&v)[16]) {
    asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
            : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
            "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
            : "r"(addr)
            : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]),
                 "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// Shared-memory matrix descriptor, 128-byte swizzle: 128-byte rows, eight to an atom, atoms `stride` bytes apart along
// the rows; `lead`: between blocks of 128-byte columns (used where the operand is N-major and wider than 64).
__device__ __forceinline__ uint64_t make_desc(uint32_t saddr, uint32_t lead, uint32_t stride) {
    return (uint64_t)((saddr & 0x3ffff) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | (uint64_t)1 << 46
            | (uint64_t)2 << 61;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// two f32 at a time
__device__ __forceinline__ uint64_t f32x2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// f16 tiles: [block of 64 dims][row][128 bytes], 16-byte pieces swizzled by the row
__device__ __forceinline__ uint32_t piece_at(int row, int piece) {
    return (uint32_t)((piece >> 3) * (UNIT * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
}

template <int DP, bool S8, bool FINE, int RUN>
__global__ void __launch_bounds__(THREADS, 1) kv_attention_tc_kernel(const __grid_constant__ b200_kv_attention_params_t p) {
    using S = smem_t<DP>;
    constexpr int CHUNKS = UNIT / RUN; // runs of a unit
    extern __shared__ uint8_t smem_raw[];
    __shared__ ctrl_t ctrl_mem;
    ctrl_t *ctrl = &ctrl_mem;
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *smem_q = smem, *smem_k = smem + 2 * S::MAT, *smem_v = smem_k + STAGES * S::MAT;
    const b200_kv_cache_t &c = p.cache;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t *status = c.status;

    part_t line;
    if (!begin_part<ROWS, EXTRA, MIN_PART>(p, line, ctrl->line_words)) return;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ctrl->q_full[i], SOFTMAX_WARPS / 2);
            for (int b = 0; b < STEPS; ++b) {
                mbar_init(&ctrl->p_full[i][b], SOFTMAX_WARPS / 2);
                mbar_init(&ctrl->s_full[i][b], 1);
                mbar_init(&ctrl->o_done[i][b], 1);
            }
        }
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&ctrl->k_full[i], CONVERT_WARPS);
            mbar_init(&ctrl->v_full[i], CONVERT_WARPS);
            mbar_init(&ctrl->k_empty[i], 2); // both issuers
            mbar_init(&ctrl->v_empty[i], 2);
        }
        for (int i = 0; i < SEGMENTS; ++i) {
            mbar_init(&ctrl->seg_full[i], 1);
            mbar_init(&ctrl->seg_empty[i], SOFTMAX_WARPS + CONVERT_WARPS + 2);
        }
        mbar_init(&ctrl->join, SOFTMAX_WARPS);
        for (int i = 0; i < 2; ++i) mbar_init(&ctrl->drained[i], 1);
        ctrl->abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctrl->tmem_base)), "r"(TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // Tensor memory columns: S_0 | S_1 | O_0 | O_1.  All 512 are this block's, so they begin at 0.
    constexpr uint32_t tmem = 0;
    const int group = line.group;
    // the segment of number i, once it is laid out (nullptr when a wait ran out); given back by every warp that took it
    auto take = [&](uint32_t i) -> const segment_t * {
        return warp_wait(&ctrl->seg_full[i % SEGMENTS], (i / SEGMENTS) & 1, ctrl, status) ? &ctrl->segments[i % SEGMENTS] : nullptr;
    };
    // steps of a segment: up to its last token, one at least
    auto steps_of = [&](const segment_t &g) { return max(1, min(g.u1 * STEPS, (g.tokens + STEP - 1) / STEP) - g.u0 * STEPS); };
    auto give_back = [&](uint32_t i) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctrl->seg_empty[i % SEGMENTS]);
    };

    if (warp < SOFTMAX_WARPS) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
        // ---------------- softmax: row r of tile t ----------------
        const int t = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tmem_s = tmem + lanes + (uint32_t)(t * UNIT), tmem_o = tmem + lanes + 2 * UNIT + (uint32_t)(t * DP);
        const bool bf16 = p.query_dt == B200_DT_BF16;
        float *parts = (float *)((char *)p.scratch + counter_bytes(gridDim.x));
        constexpr size_t part_size = (size_t)ROWS * (DP + 2);
        uint32_t s_phase = 0, o_phase = 0, tile_i = 0; // phases: a bit per place; units since the launch
        bool ok = true;
        uint32_t join_phase = 0;
        auto join = [&]() { // all softmax warps
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctrl->join);
            ok = warp_wait(&ctrl->join, join_phase, ctrl, status);
            join_phase ^= 1;
            return ok;
        };
        // the warp's query rows of a segment, as they are, into their places in shared memory; a row by DP / 8 lanes
        auto fetch = [&](const segment_t &g) {
            int64_t at = -1;
            if (t * TILE + r < g.rows) {
                const int idx = g.row0 + t * TILE + r;
                at = (int64_t)(g.begin + idx / group) * p.query_s0 + ((int64_t)g.head * group + idx % group) * p.query_s1;
            }
            constexpr int PIECES = DP / 8;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int row = i * (32 / PIECES) + lane / PIECES, piece = lane % PIECES;
                const int64_t from = __shfl_sync(~0u, at, row);
                if (from >= 0 && piece * 8 < c.dim)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem_q + t * S::MAT + piece_at((warp & 3) * 32 + row, piece))),
                                 "l"((const char *)p.query + (from + piece * 8) * 2)
                                 : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            __syncwarp(); // loads of tensor memory follow, which a warp issues together
        };
        // The row of an item that `fetch` brought: to f16 after a power of two that brings its largest element to [1, 2).
        // A negative softmax scale turns the query round, so that factors of the scores are positive.
        auto prepare = [&](bool there) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncwarp();
            uint8_t *to = smem_q + t * S::MAT;
            uint32_t top2 = 0; // the largest magnitudes' bits, of even and of odd elements
#pragma unroll 4
            for (int i = 0; i < DP / 8; ++i) {
                if (!there || i * 8 >= c.dim) *(uint4 *)(to + piece_at(r, i)) = make_uint4(0, 0, 0, 0);
                const uint4 w = *(const uint4 *)(to + piece_at(r, i));
                top2 = __vmaxu2(__vmaxu2(top2, w.x & 0x7fff7fffu), __vmaxu2(__vmaxu2(w.y & 0x7fff7fffu, w.z & 0x7fff7fffu), w.w & 0x7fff7fffu));
            }
            const float2 tops = bf16 ? bf16x2_to_f32(top2) : f16x2_to_f32(top2);
            const uint32_t top = max(__float_as_uint(tops.x), __float_as_uint(tops.y));
            const int e = top == 0 ? 127 : min(max((int)(top >> 23), 1), 253);
            float down = __uint_as_float((uint32_t)(254 - e) << 23);
            if (p.scale < 0.f) down = -down;
#pragma unroll 4
            for (int i = 0; i < DP / 8; ++i) {
                const uint4 w = *(const uint4 *)(to + piece_at(r, i));
                const uint32_t x[4] = {w.x, w.y, w.z, w.w};
                uint32_t y[4];
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const float2 f = bf16 ? bf16x2_to_f32(x[h]) : f16x2_to_f32(x[h]);
                    y[h] = pack_f16x2(f.x * down, f.y * down);
                }
                *(uint4 *)(to + piece_at(r, i)) = make_uint4(y[0], y[1], y[2], y[3]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctrl->q_full[t]);
            // the factor of the row's scores, in log2.  It times a key scale, both held to 2^-63, stays a normal number: -inf times
            // it is -inf
            return fmaxf(fabsf(p.scale) * 1.4426950408889634f * __uint_as_float((uint32_t)e << 23), SMALL);
        };
        float factor = 0.f;
        uint32_t seg_i = 0;
        const segment_t *seg = take(0);
        if (seg) {
            fetch(*seg);
            if (seg->rows > t * TILE) factor = prepare(t * TILE + r < seg->rows);
        }
        while (seg && seg->rows > 0) {
            const int u0 = seg->u0, u1 = seg->u1;
            const bool active = ok && seg->rows > t * TILE, mine = t * TILE + r < seg->rows;
            float m = -INFINITY, k2 = K_MIN, l = 0.f; // k2: k; the largest of the warp's
            // the next segment: its queries come while this one's last tile is worked on, once that one's scores are there
            const segment_t *next = nullptr;
            float factor_next = 0.f;
            auto fetch_next = [&]() {
                next = take(seg_i + 1);
                if (next) fetch(*next);
            };
            auto prepare_next = [&]() {
                if (next && next->rows > t * TILE) factor_next = prepare(t * TILE + r < next->rows);
            };
            if (active) {
                const int limit = mine ? seg->first + (seg->row0 + t * TILE + r) / group : -1;
                const int first_limit = __shfl_sync(~0u, limit, 0); // the smallest of the warp's rows that exist
                const int steps = steps_of(*seg);
                // the latest products with the weights in `place` (two may be under way, one per place)
                auto products_done = [&](int place) { return warp_wait(&ctrl->o_done[t][place], (o_phase >> place & 1) ^ 1, ctrl, status); };
                for (int j = 0; j < steps; ++j) {
                    const int place = j % STEPS;
                    if (!(ok = warp_wait(&ctrl->s_full[t][place], s_phase >> place & 1, ctrl, status))) break;
                    s_phase ^= 1u << place;
                    tc_fence_after();
                    if (j + 1 == steps) fetch_next();
                    const scales_t &sc = ctrl->scales[(tile_i + j / STEPS) & 3];
                    const float4 *chunk = sc.chunk + place * (STEP / RUN);
                    const uint32_t tmem_p = tmem_s + place * STEP;
                    // ---- the scores, and the largest
                    uint32_t v[2][32];
                    float4 ck[STEP / RUN];
#pragma unroll
                    for (int k = 0; k < STEP / RUN; ++k) ck[k] = chunk[k];
                    tmem_ld32_issue(tmem_p, v[0]);
                    tmem_ld32_issue(tmem_p + 32, v[1]);
                    tmem_ld32_wait(v[0]);
                    tmem_ld32_wait(v[1]);
                    if (u0 * UNIT + j * STEP + STEP - 1 > first_limit) { // the last steps: what a row does not see goes from its scores
                        const int seen = limit - u0 * UNIT - j * STEP;   // columns 0 .. seen are seen
#pragma unroll
                        for (int i = 0; i < STEP; ++i)
                            if (i > seen) v[i >> 5][i & 31] = 0xff800000u;
                    }
                    float f[STEP / RUN], xk[STEP / RUN], top = -INFINITY;
#pragma unroll
                    for (int k = 0; k < STEP / RUN; ++k) {
                        const uint32_t *y = v[k * RUN >> 5] + (k * RUN & 31);
                        float x0 = max3(__uint_as_float(y[0]), __uint_as_float(y[1]), __uint_as_float(y[2]));
                        float x1 = max3(__uint_as_float(y[RUN / 2]), __uint_as_float(y[RUN / 2 + 1]), __uint_as_float(y[RUN / 2 + 2]));
#pragma unroll
                        for (int i = 3; i + 1 < RUN / 2; i += 2) {
                            x0 = max3(x0, __uint_as_float(y[i]), __uint_as_float(y[i + 1]));
                            x1 = max3(x1, __uint_as_float(y[RUN / 2 + i]), __uint_as_float(y[RUN / 2 + i + 1]));
                        }
                        x0 = max3(x0, x1, __uint_as_float(y[RUN / 2 - 1]));
                        f[k] = ck[k].x * factor;
                        xk[k] = fmaf(fmaxf(x0, __uint_as_float(y[RUN - 1])), f[k], ck[k].y);
                        top = fmaxf(top, xk[k]);
                    }
                    // ---- m and k follow, seldom; O and the sum with them.  `rel`: the largest x + log2(value scale) of the step, less
                    // m (differences first, so that scores of any size keep them).  Runs of 8, twice as many, are looked at one by
                    // one where their scales are further than 2^4 apart, else the largest stands for all (24 tokens per page: 345 us, each
                    // time 350; with runs of 16 the branch costs more than it saves: 340, without 338)
                    const float from = m == -INFINITY ? top : m;
                    float rel = (top - from) + sc.above;
                    if (RUN == 16 || sc.above - sc.below > 5.f) {
                        rel = -INFINITY;
#pragma unroll
                        for (int k = 0; k < STEP / RUN; ++k) rel = fmaxf(rel, (xk[k] - from) + ck[k].z);
                    }
                    const bool follow = top > m + ROOM || rel > k2; // also from -inf
                    if (__any_sync(~0u, follow)) {
                        float fo = 1.f, d = 1.f;
                        if (follow) { // (fmaxf passes over the NaN of infinite scores)
                            const float now = fmaxf(m, top), less = m - now;
                            const float k = fminf(fmaxf(fmaxf(k2 + less, rel + (from - now) + ROOM), K_MIN), K_MAX);
                            d = fabsf(now) > M_MOST ? NAN : ex2(less), fo = ex2(less + (k2 - k));
                            m = now, k2 = k;
                        }
                        l *= d;
                        if (j > 0) { // the products of the step before are added up first
                            if (!(ok = products_done(place ^ 1))) break;
                            tc_fence_after();
#pragma unroll 1
                            for (int h = 0; h < DP / 16; ++h) {
                                uint32_t w[16];
                                tmem_ld16(tmem_o + h * 16, w);
#pragma unroll
                                for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(__uint_as_float(w[i]) * fo);
                                tmem_st16(tmem_o + h * 16, w);
                            }
                        }
                    }
                    // ---- weights, over the scores: of each 16 columns the first eight, FINE: the other eight too
                    const float base = m == -INFINITY ? 0.f : m, unit = ex2(P_TOP - k2);
#pragma unroll
                    for (int h = 0; h < STEP / 16; ++h) {
                        uint32_t pw[FINE ? 16 : 8];
#pragma unroll
                        for (int k = h * 16 / RUN; k < (h + 1) * 16 / RUN; ++k) {
                            const uint32_t *y = v[k * RUN >> 5] + (k * RUN & 31);
                            const float g = min_nan(ck[k].w * unit, G_MAX);
                            const uint64_t ff = f32x2(f[k], f[k]), oo = f32x2(ck[k].y - base, ck[k].y - base), vv = f32x2(g, g);
                            uint64_t sum = 0;
#pragma unroll
                            for (int i = 0; i < RUN; i += 2) {
                                const int at = (k * RUN % 16 + i) / 2;
                                const float2 x = unpack2(fma2(f32x2(__uint_as_float(y[i]), __uint_as_float(y[i + 1])), ff, oo));
                                const float e0 = ex2(x.x), e1 = ex2(x.y);
                                sum = add2(sum, f32x2(e0, e1));
                                const float2 pv = unpack2(mul2(f32x2(e0, e1), vv));
                                const uint32_t hi = pack_f16x2(pv.x, pv.y);
                                pw[at] = hi;
                                if (FINE) {
                                    const float2 had = f16x2_to_f32(hi);
                                    pw[FINE ? 8 + at : 0] = pack_f16x2(pv.x - had.x, pv.y - had.y);
                                }
                            }
                            const float2 both = unpack2(sum);
                            l += both.x + both.y;
                        }
                        if (FINE) tmem_st16(tmem_p + h * 16, pw);
                        else tmem_st8(tmem_p + h * 16, pw);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctrl->p_full[t][place]);
                    o_phase ^= 1u << place;
                }
                if (ok) {
                    prepare_next(); // beside the last products
                    ok = products_done((steps - 1) % STEPS);
                    tc_fence_after();
                }
            } else {
                fetch_next();
                prepare_next();
            }
            tile_i += (uint32_t)(u1 - u0);

            // ---- the row's result, or its part of it
            const bool whole = seg->whole;
            const float up = ex2(k2 - P_TOP); // O is relative to 2^(m + k - 13), parts, as l, to 2^m
            if (l != l) m = INFINITY; // a NaN among the scores, which no maximum shows
            const int idx = seg->row0 + t * TILE + r;
            char *to = (char *)p.dst + ((int64_t)(seg->begin + idx / group) * p.dst_s0 + ((int64_t)seg->head * group + idx % group) * p.dst_s1) * 2;
            auto part_of = [&](int b) { return parts + ((size_t)b * 2 + (b == seg->c0 ? 1 : 0)) * part_size; }; // place_t::part
            float *part = part_of(blockIdx.x);
            const int pr = t * TILE + r; // row of the item
            auto put = [&](int d, const float (&x)[8], float inv) { // eight dims of the result
                if (d >= c.dim) return;
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = x[i] * inv;
                store8(p.dst_dt, to + d * 2, y);
            };
            if (active && ok) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
                for (int h = 0; h < DP / 32; ++h) {
                    uint32_t v[32];
                    tmem_ld32(tmem_o + h * 32, v);
                    if (mine) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            float x[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) x[k] = __uint_as_float(v[i + k]) * up;
                            if (whole) {
                                put(h * 32 + i, x, inv);
                            } else { // rows side by side, so that a warp's stores are contiguous
                                float4 *d4 = (float4 *)(part + 2 * ROWS) + (h * 32 + i) / 4 * ROWS + pr;
                                d4[0] = make_float4(x[0], x[1], x[2], x[3]);
                                d4[ROWS] = make_float4(x[4], x[5], x[6], x[7]);
                            }
                        }
                    }
                    __syncwarp(); // the next load is the whole warp's, lanes without a row among them
                }
                tc_fence_before(); // O may be written again after the next arrival
                if (!whole && mine) part[pr] = m, part[ROWS + pr] = l;
            }
            if (!whole && ok) {
                // an item in several parts: the last block to finish one puts them together, in the order of the parts
                const int c0 = seg->c0, c1 = seg->c1;
                __threadfence();
                if (join() && threadIdx.x == 0) {
                    uint32_t *count = (uint32_t *)p.scratch + c0;
                    const bool is_last = atomicAdd(count, 1u) == (uint32_t)(c1 - c0);
                    if (is_last) *count = 0; // as it was found
                    ctrl->last_part = is_last;
                }
                if (ok && join() && ctrl->last_part && mine) {
                    __threadfence();
                    float mm = -INFINITY, ll = 0.f;
#pragma unroll 4
                    for (int b = c0; b <= c1; ++b) mm = fmaxf(mm, __ldcg(part_of(b) + pr));
#pragma unroll 4
                    for (int b = c0; b <= c1; ++b) {
                        const float mb = __ldcg(part_of(b) + pr), lb = __ldcg(part_of(b) + ROWS + pr), f = mb == -INFINITY ? 0.f : ex2(mb - mm);
                        if (f != 0.f) ll = fmaf(lb, f, ll);
                    }
                    const float inv = ll == 0.f ? 0.f : 1.f / ll;
#pragma unroll 1
                    for (int d = 0; d < DP; d += 64) {
                        float x[8][8];
#pragma unroll
                        for (int i = 0; i < 8; ++i)
#pragma unroll
                            for (int k = 0; k < 8; ++k) x[i][k] = 0.f;
#pragma unroll 1
                        for (int b = c0; b <= c1; ++b) {
                            const float4 *d4 = (const float4 *)(part_of(b) + 2 * ROWS) + d / 4 * ROWS + pr;
                            float4 y[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i) y[i] = __ldcg(d4 + i * ROWS);
                            const float mb = __ldcg(part_of(b) + pr), f = mb == -INFINITY ? 0.f : ex2(mb - mm);
                            if (f == 0.f) continue;
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                float *z = x[i / 2] + (i & 1) * 4;
                                z[0] = fmaf(y[i].x, f, z[0]), z[1] = fmaf(y[i].y, f, z[1]), z[2] = fmaf(y[i].z, f, z[2]), z[3] = fmaf(y[i].w, f, z[3]);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i) put(d + i * 8, x[i], inv);
                    }
                }
            }
            give_back(seg_i++);
            seg = next;
            factor = factor_next;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else if (warp < MMA_WARP) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CONVERT_REGS));
        // ---------------- codes to f16 ----------------
        // Warp w has tokens 32 w .. of a tile: runs of RUN, each in one page.  An access of the warp covers 512 / DP tokens in
        // groups of eight lanes: two tokens, 64 dims each, so that both the 64-byte reads and the stores (pieces
        // 0, 2, 4, 6 of an even token, swizzled, and of the odd one next to it) use all that they touch.
        constexpr int CH = DP / 16, PER = 32 / CH, LOADS = 32 / PER;
        const int w = warp - SOFTMAX_WARPS, page = (int)c.page;
        const int cc = DP == 64 ? lane & 3 : (lane & 3) + (lane >> 3 & 1) * 4; // 16 codes of a token
        const int sub_row = DP == 64 ? lane >> 2 : (lane >> 4) * 2 + (lane >> 2 & 1);
        const bool takes = cc * 16 < c.dim;
        const int64_t lane_at = sub_row * c.s_slot, per_step = PER * c.s_slot;
        uint32_t tile_i = 0, seg_i = 0;
        bool ok = true;
        while (ok) {
            const segment_t *seg = take(seg_i);
            if (!seg || seg->rows == 0) break;
            const int u0 = seg->u0, u1 = seg->u1, end = seg->tokens, head = seg->head;
            if (w == 0 && lane == 0 && u0 == 0 && seg->over) flag_bad_page(c);
            const int32_t *table = c.table + (int64_t)seg->seq * c.table_s0;
            give_back(seg_i++);
            const uint8_t *keys = (const uint8_t *)c.key + head * c.s_head + cc * 16, *values = (const uint8_t *)c.value + head * c.s_head + cc * 16;
            uint4 kr[LOADS], vr[LOADS];
            // every warp looks up all runs of a tile, one per lane
            int64_t place = -1;
            float ks = -1.f, vs = 0.f;
            int n = (u0 * UNIT + lane * RUN) / page, slot = u0 * UNIT + lane * RUN - n * page;
            const int jump_n = UNIT / page, jump_slot = UNIT - jump_n * page;
            auto find = [&](int j) {
                place = -1, ks = -1.f, vs = 0.f;
                if (lane < CHUNKS && j < u1 && j * UNIT + lane * RUN < end) {
                    const int phys = table[n];
                    if (phys >= 0 && phys < c.pages) {
                        place = (int64_t)phys * c.s_page + (int64_t)slot * c.s_slot;
                        const int64_t i = (int64_t)phys * c.heads + head;
                        ks = c.key_scale[i], vs = c.value_scale[i];
                    } else {
                        flag_bad_page(c);
                    }
                }
                n += jump_n, slot += jump_slot;
                if (slot >= page) slot -= page, ++n;
            };
            auto load = [&](int j, const uint8_t *from, uint4 (&regs)[LOADS]) {
                int64_t run[32 / RUN], worst = 0;
#pragma unroll
                for (int k = 0; k < 32 / RUN; ++k) {
                    run[k] = __shfl_sync(~0u, place, w * (32 / RUN) + k);
                    worst |= run[k];
                }
                const int left = end - j * UNIT - w * 32;
                static_assert(RUN % PER == 0, "an access stays in its run");
                if (DP == c.dim && worst >= 0 && left >= 32) { // all there
#pragma unroll
                    for (int i = 0; i < LOADS; ++i) // a run's accesses are PER tokens apart
                        regs[i] = __ldg((const uint4 *)(from + run[i * PER / RUN] + lane_at + (i % (RUN / PER)) * per_step));
                    return;
                }
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const int tok = i * PER + sub_row; // of the warp's 32; the run is known at compile time
                    regs[i] = make_uint4(0, 0, 0, 0);
                    if (takes && run[i * PER / RUN] >= 0 && tok < left)
                        regs[i] = __ldg((const uint4 *)(from + run[i * PER / RUN] + (tok & (RUN - 1)) * c.s_slot));
                }
            };
            auto convert = [&](const uint4 (&regs)[LOADS], uint8_t *to) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const int row = w * 32 + i * PER + sub_row;
                    uint4 a, b;
                    widen<S8>(regs[i].x, a.x, a.y);
                    widen<S8>(regs[i].y, a.z, a.w);
                    widen<S8>(regs[i].z, b.x, b.y);
                    widen<S8>(regs[i].w, b.z, b.w);
                    *(uint4 *)(to + piece_at(row, cc * 2)) = a;
                    *(uint4 *)(to + piece_at(row, cc * 2 + 1)) = b;
                }
            };
            // keys of unit j (the i-th since the launch), and both scales: a softmax that sees the scores sees them
            auto put_keys = [&](uint32_t i) {
                const int st = i % STAGES;
                const uint32_t use = i / STAGES;
                if (use > 0 && !(ok = warp_wait(&ctrl->k_empty[st], (use - 1) & 1, ctrl, status))) return;
                if (w == 0) {
                    const bool there = ks >= 0.f;
                    // scales are positive, so their bits compare like them
                    const uint32_t bits = __float_as_uint(vs), vmax = __reduce_max_sync(~0u, there ? bits : 0u);
                    const uint32_t vmin = min(__reduce_min_sync(~0u, there ? bits : ~0u), vmax);
                    scales_t &sc = ctrl->scales[i & 3];
                    const float above = (float)((int)(bits >> 23) - 126);
                    if (lane < CHUNKS) sc.chunk[lane] = there ? make_float4(fmaxf(ks, SMALL), 0.f, above, vs) : make_float4(SMALL, -INFINITY, 0.f, 0.f);
                    if (lane == 0) sc.above = (float)((int)(vmax >> 23) - 126), sc.below = (float)((int)(vmin >> 23) - 127);
                }
                convert(kr, smem_k + st * S::MAT);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->k_full[st]);
            };
            // the keys go a unit ahead of the values: the scores are computed that much ahead of the products
            find(u0);
            load(u0, keys, kr);
            load(u0, values, vr);
            put_keys(tile_i);
            find(u0 + 1);
            load(u0 + 1, keys, kr);
            for (int j = u0; j < u1 && ok; ++j, ++tile_i) {
                if (j + 1 < u1) put_keys(tile_i + 1);
                if (!ok) break;
                const int st = tile_i % STAGES;
                const uint32_t use = tile_i / STAGES;
                if (use > 0 && !(ok = warp_wait(&ctrl->v_empty[st], (use - 1) & 1, ctrl, status))) break;
                convert(vr, smem_v + st * S::MAT);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->v_full[st]);
                load(j + 1, values, vr);
                find(j + 2);
                load(j + 2, keys, kr);
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(MMA_REGS));
        // ---------------- the MMAs ----------------
        // The whole warp walks through the loops, so that descriptors and addresses are uniform values; one lane
        // issues.  Tensor memory addresses are constants: the kernel allocates all columns.
        constexpr uint32_t IDESC = (1u << 4) | ((uint32_t)(TILE >> 4) << 24);
        constexpr uint32_t IDESC_S = IDESC | ((uint32_t)(STEP >> 3) << 17);
        constexpr uint32_t IDESC_O = IDESC | (1u << 16) | ((uint32_t)(DP >> 3) << 17); // values are N-major
        const uint64_t q_desc = make_desc(smem_u32(smem_q), 16, 1024), k_desc = make_desc(smem_u32(smem_k), 16, 1024);
        const uint64_t v_desc = make_desc(smem_u32(smem_v), UNIT * 128, 1024);
        const int t = warp - MMA_WARP; // 0, 1: the tile
        uint32_t q_phase = 0, p_phase = 0, tile_i = 0, seg_i = 0; // p_phase: a bit per place
        bool ok = true;
        auto scores = [&](int st, int place) { // S_t = Q_t K^T, the place's half of a unit
            const uint64_t a = q_desc + (uint64_t)(t * (S::MAT >> 4)), b = k_desc + (uint64_t)((st * S::MAT + place * STEP * 128) >> 4);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
                    const uint32_t o = (uint32_t)((k >> 2) * (UNIT * 128) + (k & 3) * 32) >> 4;
                    mma_ss(t * UNIT + place * STEP, a + o, b + o, IDESC_S, k != 0);
                }
                tc_commit(&ctrl->s_full[t][place]);
            }
        };
        auto weigh = [&](int st, int place, bool more) { // O_t += P_t V
            const uint64_t b = v_desc + (uint64_t)((st * S::MAT + place * STEP * 128) >> 4);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < STEP / 16; ++k) {
                    const uint32_t a = t * UNIT + place * STEP + k * 16;
                    mma_ts(2 * UNIT + t * DP, a, b + k * (2048 >> 4), IDESC_O, more || k != 0);
                    if (FINE) mma_ts(2 * UNIT + t * DP, a + 8, b + k * (2048 >> 4), IDESC_O, 1);
                }
                tc_commit(&ctrl->o_done[t][place]);
            }
        };
        auto commit = [&](uint64_t *bar) {
            if (elect_one()) tc_commit(bar);
        };
        while (t < 2 && ok) {
            const segment_t *seg = take(seg_i);
            if (!seg || seg->rows == 0) break;
            const int n = steps_of(*seg), units = seg->u1 - seg->u0;
            const bool active = seg->rows > t * TILE;
            give_back(seg_i++);
            auto stage = [&](int s) { return (int)((tile_i + s / STEPS) % STAGES); };
            auto use = [&](int s) { return (tile_i + s / STEPS) / STAGES & 1; };
            auto wait = [&](uint64_t *bar, uint32_t parity) { return ok = warp_wait(bar, parity, ctrl, status); };
            if (!active) { // no rows in this tile: the stages are given back as they come
                for (int s = 0; s < n; s += STEPS) {
                    if (!wait(&ctrl->k_full[stage(s)], use(s))) break;
                    if (lane == 0) mbar_arrive(&ctrl->k_empty[stage(s)]);
                    if (!wait(&ctrl->v_full[stage(s)], use(s))) break;
                    if (lane == 0) mbar_arrive(&ctrl->v_empty[stage(s)]);
                }
                tile_i += (uint32_t)units;
                continue;
            }
            if (!wait(&ctrl->k_full[stage(0)], use(0)) || !wait(&ctrl->q_full[t], q_phase)) break;
            q_phase ^= 1;
            tc_fence_after();
            scores(stage(0), 0);
            if (n > 1) scores(stage(0), 1);
            commit(&ctrl->k_empty[stage(0)]);
            for (int s = 0; s < n; ++s) {
                const int place = s % STEPS;
                if (place == 0) {
                    if (!wait(&ctrl->v_full[stage(s)], use(s))) break;
                    if (s + 2 < n && !wait(&ctrl->k_full[stage(s + 2)], use(s + 2))) break;
                }
                if (!wait(&ctrl->p_full[t][place], p_phase >> place & 1)) break;
                p_phase ^= 1u << place;
                tc_fence_after();
                weigh(stage(s), place, s > 0);
                if (place == 1 || s + 1 == n) commit(&ctrl->v_empty[stage(s)]);
                if (s + 2 < n) {
                    scores(stage(s + 2), place);
                    if (place == 1 || s + 3 == n) commit(&ctrl->k_empty[stage(s + 2)]);
                }
            }
            tile_i += (uint32_t)units;
        }
        if (t == 2) {
            // ---------------- the segments ----------------
            int64_t at = line.begin;
            for (uint32_t i = 0;; ++i) {
                segment_t g;
                g.rows = 0;
                while (at < line.stop && g.rows == 0) {
                    const place_t q = find_item<ROWS, EXTRA>(p, line, at);
                    at = q.next;
                    if (q.u1 <= q.u0) continue; // the block has none of its tokens
                    g.begin = line.s.begin;
                    g.row0 = q.tile * ROWS;
                    g.rows = (line.s.end - line.s.begin) * group - g.row0;
                    g.first = line.s.first;
                    g.head = q.head;
                    g.seq = line.seq;
                    g.tokens = q.item.tokens;
                    g.u0 = q.u0;
                    g.u1 = q.u1;
                    g.whole = q.whole();
                    g.c0 = q.c0;
                    g.c1 = q.c1;
                    g.over = (int64_t)line.s.first + (line.s.end - line.s.begin) > line.capacity;
                }
                const bool more = g.rows > 0;
                if (i >= SEGMENTS && !warp_wait(&ctrl->seg_empty[i % SEGMENTS], (i / SEGMENTS - 1) & 1, ctrl, status)) break;
                if (lane == 0) {
                    ctrl->segments[i % SEGMENTS] = g;
                    mbar_arrive(&ctrl->seg_full[i % SEGMENTS]);
                }
                __syncwarp();
                if (!more) break;
            }
        }
    }
    // All roles are through.  The MMAs too, every one was waited for by way of o_done -- unless a wait ran out: then their
    // issuers wait for what is still under way, before its operands and results are given up.
    __syncthreads();
    if (ctrl->abort) {
        if (warp == MMA_WARP || warp == MMA_WARP + 1) {
            uint64_t *bar = &ctrl->drained[warp - MMA_WARP];
            if (elect_one()) tc_commit(bar);
            __syncwarp();
            const uint64_t until = now_ns() + WAIT_NS;
            for (uint32_t i = 0; i < WAIT_TRIES && !mbar_try(bar, 0); ++i)
                if ((i & 255) == 255 && now_ns() > until) break;
        }
        __syncthreads();
    }
    if (warp == MMA_WARP) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

template <int DP, bool S8, bool FINE, int RUN>
int run(const b200_kv_attention_params_t &p, cudaStream_t cs) {
    auto kernel = kv_attention_tc_kernel<DP, S8, FINE, RUN>;
    const int bytes = smem_t<DP>::BYTES + 1024;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return (int)e;
    kernel<<<p.sm_count, THREADS, bytes, cs>>>(p);
    return after_launch();
}
template <int DP, bool S8, bool FINE>
int run(const b200_kv_attention_params_t &p, cudaStream_t cs) {
    return p.cache.page % 16 == 0 ? run<DP, S8, FINE, 16>(p, cs) : run<DP, S8, FINE, 8>(p, cs);
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
    // what the other kernel takes, with pages of whole runs of 8 tokens
    if (!b200_kv_attention_mma_supported(p) || p->cache.dim > 128 || p->cache.page % 8) return 0;
    // and at least 48 query rows per sequence and key head: a tile costs the same however many of its rows there are.  16
    // sequences of 700 to 4500 tokens, 8 query heads on each of 5 key heads: there 32 rows take 52 us, 48 62, 64 76, 128 134;
    // here 48 to 128 take 64.
    return p->cache.seqs > 0 && p->cache.heads > 0 && p->rows / p->cache.seqs * (p->q_heads / p->cache.heads) >= 48;
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
