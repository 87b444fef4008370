// Attention over the paged 8-bit cache for few query rows per key head (b200_kv_attention_mma_launch): steps of one
// token, drafts of a few.  Bound by reading the cache once.
//
// Work items of up to 8 * NB query rows are laid out and cut as kv_line.cuh says, so that ragged batches and
// single long contexts load every SM alike.  An item that was cut is put together by the block that
// finishes it last, in the order of the parts, so the result does not depend on who is last.
//
// Inside a block each of four warps takes every fourth 32 tokens through a ring of its own in shared memory (cp.async,
// no block barrier in the loop) with its own running maximum, sum and weighted values:
//   S^T (tokens x rows) = K Q^T,  O^T (dim x rows) = V^T P^T      mma.m16n8k16, f16 in, f32 out
// Tokens and dims sit on the 16-wide side, so eight query rows already fill the instruction.  The codes become
// f16 exactly (both types fit) in registers; which dim or token an instruction's k index stands for is free as
// long as both operands agree, so the fragments are chosen to be 16-byte pieces of the rows as they lie in the cache.
// FINE (f16 results): what a weight's rounding to f16 left is multiplied too; bf16's own last rounding is eight
// times as large, so there it would not show.
// Scales stay out of the products: the key's multiplies the score, the value's the weight.  f16 holds weight times
// value scale, P = 2^(x - m) * 2^(14 - k) * scale, with two numbers of each row: m, the largest score x that it has seen, and k, such
// that no token that it sees has x + log2(scale) above m + k (k goes down as m goes up, exactly: rounded to whole numbers it
// stayed, and scores that rose by less than 2 per step left m + k far above all that counted).  So P < 2^14, rounded to 2^-11 of
// itself down to 2^-28 of that, and no page that a row does not see, or gives no weight, takes bits from the others.  In a
// step whose scales lie within 2^4 of one another the largest stands for all; else k comes from the tokens one by one.
// The sum is relative to 2^m, the weighted values to 2^(m + k - 14).  Queries are taken to f16 after a power of two per row that
// brings the largest element to [1, 2).
#pragma once

#include "kv_f16.cuh"
#include "kv_line.cuh"
#include "launch.hpp"

#include <type_traits>

//
// Measured on one B200: 64 sequences of 900 to 8100 tokens, 32 query heads on 8, dim 128: s8 120 us, e4m3 112 us (574 MB: 4.8
// and 5.1 TB/s); one of 131009 tokens: 65 us (4.1 TB/s).  Some 900 instructions per 32 tokens and warp at 0.5 per
// cycle and scheduler: three blocks of four warps per SM are what registers and rings allow (two blocks: 150 us), and
// the loops wait for their own results more than for memory.
namespace b200 {
namespace kv_mma {

using namespace kv_line;

constexpr int EXTRA = 1; // units that an item's queries and result take besides
constexpr int WARPS = 4, THREADS = WARPS * 32, STEP = 32;
constexpr float P_TOP = 14.f; // weights in f16 stay below 2^14
constexpr float K_MIN = -100.f, K_MAX = 121.f; // of k: where all scales that a row sees are below 2^-100, f16's last bits go unused
static_assert(WARPS * STEP == UNIT, "a warp takes one step of each unit");

// blocks per SM
__host__ __device__ constexpr int blocks_of(int dp, int nb) { return dp == 64 ? (nb == 1 ? 4 : 3) : dp == 128 ? (nb == 1 ? 3 : 2) : 1; }

template <int DP, int NB>
struct shape_t {
    static constexpr int BLOCKS = blocks_of(DP, NB);
    static constexpr int STAGES = DP == 64 ? 3 : BLOCKS == 3 ? 2 : 3;
    static constexpr int ROWS = 8 * NB;
    static constexpr int STAGE = 2 * (STEP * DP + STEP * 4);        // keys and their scales, values and theirs
    static constexpr int RING = STAGES * STAGE;
    static constexpr int PITCH = DP + 4;                            // of a row of partial values, f32
    static constexpr bool Q_SHARED = NB * DP > 256;                 // query fragments do not fit the registers
    static constexpr int Q_BYTES = Q_SHARED ? (DP / 16) * NB * 32 * 8 : 0;
    static constexpr int SMEM = WARPS * RING + Q_BYTES;
    static_assert(ROWS * PITCH * 4 <= RING, "the partial values reuse the ring");
};

inline size_t part_floats(int dp, int nb) { return (size_t)8 * nb * (dp + 2); }

// ---- small pieces -------------------------------------------------------------------------------

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool take) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// a whole number above the base-2 logarithm of a value with these bits, by one at most
__device__ __forceinline__ float above_log2(uint32_t bits) { return (float)((int)(bits >> 23) - 126); }
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) { return __byte_perm(a, b, s); }
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Where 16-byte piece `c` of token `r` lies in its row.  Eight neighbouring lanes read, of the keys, pieces t = 0..3 of two
// tokens r, r + 1; of the values, pieces g, g + 1 of the four tokens r, r + 2, r + 4, r + 6: all in different banks.
template <int DP>
__device__ __forceinline__ int key_piece(int r, int c) { return DP == 64 ? c : c ^ ((r & 1) << 2); }
template <int DP>
__device__ __forceinline__ int value_piece(int r, int c) { return DP == 64 ? c ^ (r & 2) : c ^ (r & 6); }

template <int DP, int NB, bool S8, bool RUNS, bool FINE>
__global__ void __launch_bounds__(THREADS, shape_t<DP, NB>::BLOCKS)
kv_attention_mma_kernel(const __grid_constant__ b200_kv_attention_params_t p) {
    using S = shape_t<DP, NB>;
    constexpr int ROWS = S::ROWS, KS = DP / 16, CH = DP / 16, MT = DP / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t line_words[LINE_WORDS];
    __shared__ float merge_m[WARPS][ROWS], merge_l[WARPS][ROWS];
    __shared__ bool last_part;

    const b200_kv_cache_t &c = p.cache;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    part_t line;
    if (!begin_part<ROWS, EXTRA, 1>(p, line, line_words)) return;
    const int heads = line.heads, group = line.group, page = (int)c.page, pieces = (int)c.dim / 16;
    uint8_t *ring = smem + warp * S::RING;
    uint2 *q_shared = (uint2 *)(smem + WARPS * S::RING);
    // pieces behind dim stay zero: no copy writes them
    if (pieces < CH) {
        for (int i = tid; i < WARPS * S::RING / 16; i += THREADS) ((uint4 *)smem)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }

    uint32_t *counters = (uint32_t *)p.scratch;
    float *parts = (float *)((char *)p.scratch + counter_bytes(gridDim.x));
    constexpr size_t part_size = (size_t)ROWS * (DP + 2); // part_floats()
    int64_t at = line.begin;
    while (at < line.stop) {
        const place_t place_at = find_item<ROWS, EXTRA>(p, line, at);
        at = place_at.next;
        const int u0 = place_at.u0, u1 = place_at.u1;
        if (u1 <= u0) continue; // none of its tokens
        const item_t item = place_at.item;
        const int head = place_at.head, tile = place_at.tile, seq = line.seq;
        const seq_t s = line.s;
        const int rows = (s.end - s.begin) * group - tile * ROWS; // that exist from here on
        const int end = min(u1 * UNIT, item.tokens);
        if (tid == 0 && u0 == 0 && (int64_t)s.first + (s.end - s.begin) > line.capacity) flag_bad_page(c);

        const int32_t *table = c.table + (int64_t)seq * c.table_s0;
        const uint8_t *keys = (const uint8_t *)c.key + head * c.s_head, *values = (const uint8_t *)c.value + head * c.s_head;

        // ---- copies; a lane looks a token's page up one step ahead of the copy that needs it.
        // Lane l copies piece l % CH of the CH tokens from l / CH * CH on, and its own token's scales.
        // With RUNS these tokens lie in one page, so that one place serves the lane's copies; without, every token
        // has a place of its own, from the lane that looked it up.
        const int lead = RUNS ? lane / CH * CH : lane; // the token of a step that this lane looks up
        int next_page = -1, next_j, next_slot;
        const int jump_j = UNIT / page, jump_slot = UNIT - jump_j * page;
        // steps behind the last one are left out by their number: a token of theirs may not fit 32 bits
        const int first_step = u0 * WARPS + warp, steps_end = (end + STEP - 1) / STEP;
        auto look_up_at = [&](int step) {
            next_page = -1, next_j = 0, next_slot = 0;
            if (step >= steps_end) return;
            const int tok = step * STEP + lead;
            next_j = tok / page;
            next_slot = tok - next_j * page;
            if (tok < end) next_page = table[next_j];
        };
        auto look_up_next = [&](int step) { // the warp's step after the one looked up before
            next_page = -1;
            if (step >= steps_end) return;
            next_j += jump_j;
            next_slot += jump_slot;
            if (next_slot >= page) next_slot -= page, ++next_j;
            if (step * STEP + lead < end) next_page = table[next_j];
        };
        int64_t place = -1; // of the lane's tokens in the step that is being copied
        int place_page = 0;
        bool simple = false; // all tokens are there, and rows lie densely: addresses are constants apart
        auto find = [&](int step) {
            place = -1;
            place_page = next_page;
            if (step * STEP + lead < end) {
                if (next_page >= 0 && next_page < c.pages) place = (int64_t)next_page * c.s_page + (int64_t)next_slot * c.s_slot;
                else flag_bad_page(c);
            }
            if (RUNS) simple = __all_sync(~0u, place >= 0) && (step + 1) * STEP <= end && c.s_slot == DP && c.dim == DP;
        };
        // keys (VAL false) or values of a step into a half stage, their scales behind them
        auto copy = [&](auto val, int step, uint8_t *to) {
            constexpr bool VAL = decltype(val)::value;
            const uint8_t *from = VAL ? values : keys;
            float *scales = (float *)(to + STEP * DP);
            const int left = end - step * STEP; // tokens of this step and behind
            if (RUNS && simple) {
                cp4(smem_u32(scales + lane), (VAL ? c.value_scale : c.key_scale) + (int64_t)place_page * heads + head);
                const uint8_t *f = from + place + lane % CH * 16;
                const uint32_t d = smem_u32(to + lead * DP);
#pragma unroll
                for (int i = 0; i < CH; ++i) cp16(d + i * DP + (VAL ? value_piece<DP>(i, lane % CH) : key_piece<DP>(i, lane % CH)) * 16, f + i * DP);
                return;
            }
            if (place >= 0 && lane < left) cp4(smem_u32(scales + lane), (VAL ? c.value_scale : c.key_scale) + (int64_t)place_page * heads + head);
            else scales[lane] = VAL ? 0.f : -1.f; // no such token
            const int cc = lane % CH;
            if (RUNS) {
                if (cc < pieces) {
                    const uint8_t *f = from + max(place, (int64_t)0) + cc * 16;
                    const int ok = place >= 0 ? left - lead : 0;
                    const uint32_t d = smem_u32(to + lead * DP);
#pragma unroll
                    for (int i = 0; i < CH; ++i) {
                        const bool take = i < ok; // else: no address behind the last page
                        cp16(d + i * DP + (VAL ? value_piece<DP>(i, cc) : key_piece<DP>(i, cc)) * 16, f + (take ? i * c.s_slot : 0), take);
                    }
                }
            } else {
                constexpr int PER = 32 / CH; // tokens per access of the warp
#pragma unroll
                for (int i = 0; i < STEP / PER; ++i) {
                    const int r = i * PER + lane / CH;
                    const int64_t o = __shfl_sync(~0u, place, r);
                    if (cc < pieces)
                        cp16(smem_u32(to + r * DP + (VAL ? value_piece<DP>(r, cc) : key_piece<DP>(r, cc)) * 16),
                                from + max(o, (int64_t)0) + cc * 16, o >= 0);
                }
            }
        };
        constexpr std::integral_constant<bool, false> KEYS;
        constexpr std::integral_constant<bool, true> VALUES;
#pragma unroll
        for (int i = 0; i < S::STAGES; ++i) {
            const int step = first_step + i * WARPS;
            uint8_t *k = ring + i * S::STAGE;
            if (step < steps_end) {
                look_up_at(step);
                find(step);
                copy(KEYS, step, k);
            }
            cp_commit();
            if (step < steps_end) copy(VALUES, step, k + S::STAGE / 2);
            cp_commit();
        }
        look_up_at(first_step + S::STAGES * WARPS);

        // ---- queries: row g of each tile of eight, four neighbouring dims per instruction
        uint32_t q[S::Q_SHARED ? 1 : KS][S::Q_SHARED ? 1 : NB][2];
        float factor[NB][2]; // of the scores of rows 2t, 2t + 1, in units of log2
        int limit[NB][2];    // the newest token that they see
        {
            float unit[NB];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const int r = nb * 8 + g;
                const bool mine = r < rows;
                const int idx = tile * ROWS + (mine ? r : 0);
                const int64_t off = (int64_t)(s.begin + idx / group) * p.query_s0 + (int64_t)(head * group + idx % group) * p.query_s1;
                const char *row = (const char *)p.query + off * 2;
                uint32_t w[KS][2];
                uint32_t top = 0;
                const bool bf16 = p.query_dt == B200_DT_BF16;
#pragma unroll
                for (int j = 0; j < KS / 4; ++j) {
                    uint4 a[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
                    if (mine && j * 4 + t < pieces) {
                        a[0] = *(const uint4 *)(row + (j * 64 + t * 16) * 2);
                        a[1] = *(const uint4 *)(row + (j * 64 + t * 16 + 8) * 2);
                    }
                    const uint32_t x[8] = {a[0].x, a[0].y, a[0].z, a[0].w, a[1].x, a[1].y, a[1].z, a[1].w};
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        w[j * 4 + i / 2][i & 1] = x[i];
                        const float2 f = bf16 ? bf16x2_to_f32(x[i]) : f16x2_to_f32(x[i]);
                        top = max(top, max(__float_as_uint(fabsf(f.x)), __float_as_uint(fabsf(f.y))));
                    }
                }
                top = max(top, __shfl_xor_sync(~0u, top, 1));
                top = max(top, __shfl_xor_sync(~0u, top, 2));
                // 2^e next below the largest element, 1 for a row of zeros; both 2^e and 2^-e stay normal
                int e = (int)(top >> 23);
                e = top == 0 ? 127 : min(max(e, 1), 253);
                unit[nb] = __uint_as_float((uint32_t)e << 23);
                const float down = __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    uint32_t b[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float2 f = bf16 ? bf16x2_to_f32(w[i][h]) : f16x2_to_f32(w[i][h]);
                        b[h] = pack_f16x2(f.x * down, f.y * down);
                    }
                    if (S::Q_SHARED) {
                        if (warp == 0) q_shared[(i * NB + nb) * 32 + lane] = make_uint2(b[0], b[1]);
                    } else {
                        q[i % (S::Q_SHARED ? 1 : KS)][nb % (S::Q_SHARED ? 1 : NB)][0] = b[0];
                        q[i % (S::Q_SHARED ? 1 : KS)][nb % (S::Q_SHARED ? 1 : NB)][1] = b[1];
                    }
                }
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = 2 * t + h; // of this tile of eight; lane 4 r holds its unit
                    factor[nb][h] = p.scale * 1.4426950408889634f * __shfl_sync(~0u, unit[nb], 4 * r);
                    limit[nb][h] = nb * 8 + r < rows ? s.first + (tile * ROWS + nb * 8 + r) / group : -1;
                }
        }
        if (S::Q_SHARED) __syncthreads();
        int all_see = 0x7fffffff; // up to this token no row of the item is masked
        if (rows > 0) all_see = s.first + (tile * ROWS) / group;

        float o[MT][NB][4], m[NB][2], k2[NB][2], l[NB][2]; // k2: k
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            m[nb][0] = m[nb][1] = -INFINITY;
            k2[nb][0] = k2[nb][1] = K_MIN;
            l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
            for (int i = 0; i < MT; ++i) o[i][nb][0] = o[i][nb][1] = o[i][nb][2] = o[i][nb][3] = 0.f;
        }

        int stage = 0;
        for (int step = first_step; step < steps_end; step += WARPS) {
            // later groups than these keys: values and keys of every stage but this one, and these values
            cp_wait<2 * S::STAGES - 1>();
            __syncwarp();
            uint8_t *k = ring + stage * S::STAGE, *v = k + S::STAGE / 2;
            const float *sk = (const float *)(k + STEP * DP), *sv = (const float *)(v + STEP * DP);

            // ---- scores
            float st[2][NB][4];
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) st[tt][nb][0] = st[tt][nb][1] = st[tt][nb][2] = st[tt][nb][3] = 0.f;
                const int r = tt * 16 + g;
#pragma unroll
                for (int j = 0; j < KS / 4; ++j) {
                    const uint4 x = *(const uint4 *)(k + r * DP + key_piece<DP>(r, j * 4 + t) * 16);
                    const uint4 y = *(const uint4 *)(k + (r + 8) * DP + key_piece<DP>(r + 8, j * 4 + t) * 16);
                    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t a[4];
                        widen<S8>(xs[i], a[0], a[2]);
                        widen<S8>(ys[i], a[1], a[3]);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            if (S::Q_SHARED) {
                                const uint2 u = q_shared[((j * 4 + i) * NB + nb) * 32 + lane];
                                const uint32_t b[2] = {u.x, u.y};
                                mma(st[tt][nb], a, b);
                            } else {
                                mma(st[tt][nb], a, q[(j * 4 + i) % (S::Q_SHARED ? 1 : KS)][nb % (S::Q_SHARED ? 1 : NB)]);
                            }
                        }
                    }
                }
            }
            float ks[4], vs[4]; // of tokens g, g + 8, g + 16, g + 24
#pragma unroll
            for (int i = 0; i < 4; ++i) ks[i] = sk[g + 8 * i];
            // the keys are read: their place is taken by those of STAGES steps further on
            __syncwarp();
            const int further = step + S::STAGES * WARPS;
            if (further < steps_end) {
                find(further);
                copy(KEYS, further, k);
            }
            cp_commit();
            const bool gaps = __any_sync(~0u, fminf(fminf(ks[0], ks[1]), fminf(ks[2], ks[3])) < 0.f);
            const bool masked = gaps || step * STEP + STEP - 1 > all_see;
            float top[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                top[nb][0] = top[nb][1] = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float &x = st[i >> 1][nb][(i & 1) * 2 + h];
                        x = x * ks[i] * factor[nb][h];
                    }
            }
            if (masked) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            if (ks[i] < 0.f || step * STEP + g + 8 * i > limit[nb][h]) st[i >> 1][nb][(i & 1) * 2 + h] = -INFINITY;
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) top[nb][h] = fmaxf(top[nb][h], st[i >> 1][nb][(i & 1) * 2 + h]);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) top[nb][h] = fmaxf(top[nb][h], __shfl_xor_sync(~0u, top[nb][h], w));
            cp_wait<2 * S::STAGES - 1>();
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) vs[i] = sv[g + 8 * i];
            // the largest and the smallest value scale (scales are positive, so their bits compare like them; 0: no such token)
            uint32_t vb[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) vb[i] = __float_as_uint(vs[i]);
            const uint32_t vmax = __reduce_max_sync(~0u, max(max(vb[0], vb[1]), max(vb[2], vb[3])));
            const uint32_t vmin = __reduce_min_sync(~0u, min(min(vb[0] - 1, vb[1] - 1), min(vb[2] - 1, vb[3] - 1)));
            // `now`: the largest score with this step; `rel`: the largest x + log2(scale) of the step's tokens, or up to 5 more,
            // less `now` (differences first, so that scores of any size keep them)
            float now[NB][2], rel[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    now[nb][h] = fmaxf(m[nb][h], top[nb][h]);
                    rel[nb][h] = (top[nb][h] - now[nb][h]) + above_log2(vmax);
                }
            if (vmax > 0 && (vmax >> 23) > (vmin >> 23) + 4) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float &y = rel[nb][h];
                        y = -INFINITY;
#pragma unroll
                        for (int i = 0; i < 4; ++i) y = fmaxf(y, (st[i >> 1][nb][(i & 1) * 2 + h] - now[nb][h]) + above_log2(vb[i]));
#pragma unroll
                        for (int w = 4; w < 32; w <<= 1) y = fmaxf(y, __shfl_xor_sync(~0u, y, w));
                    }
            }
            bool grew = false;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int h = 0; h < 2; ++h) grew |= now[nb][h] > m[nb][h] || rel[nb][h] > k2[nb][h];
            if (__any_sync(~0u, grew)) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    float fo[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        // (fmaxf passes over the NaN of infinite scores, or of none)
                        const float less = m[nb][h] - now[nb][h];
                        const float k = fminf(fmaxf(fmaxf(k2[nb][h] + less, rel[nb][h]), K_MIN), K_MAX);
                        fo[h] = now[nb][h] == -INFINITY ? 1.f : ex2(less + (k2[nb][h] - k));
                        l[nb][h] *= now[nb][h] == -INFINITY ? 1.f : ex2(less);
                        m[nb][h] = now[nb][h];
                        k2[nb][h] = k;
                    }
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        o[i][nb][0] *= fo[0];
                        o[i][nb][1] *= fo[1];
                        o[i][nb][2] *= fo[0];
                        o[i][nb][3] *= fo[1];
                    }
                }
            }

            // ---- weights, and the weighted values
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                uint32_t pb[NB][2], rest[NB][2];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    const float m0 = m[nb][0] == -INFINITY ? 0.f : m[nb][0], m1 = m[nb][1] == -INFINITY ? 0.f : m[nb][1];
                    const float r0 = ex2(P_TOP - k2[nb][0]), r1 = ex2(P_TOP - k2[nb][1]);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float w0 = ex2(st[tt][nb][i * 2] - m0), w1 = ex2(st[tt][nb][i * 2 + 1] - m1);
                        l[nb][0] += w0;
                        l[nb][1] += w1;
                        const float p0 = w0 * r0 * vs[tt * 2 + i], p1 = w1 * r1 * vs[tt * 2 + i]; // in this order: no weight times a large scale is 0
                        const uint32_t hi = pack_f16x2(p0, p1);
                        pb[nb][i] = transposed(hi);
                        if (FINE) {
                            const float2 had = f16x2_to_f32(hi);
                            rest[nb][i] = transposed(pack_f16x2(p0 - had.x, p1 - had.y));
                        }
                    }
                }
                const int r = tt * 16 + 2 * t; // this lane's tokens: r, r + 1, r + 8, r + 9
#pragma unroll
                for (int j = 0; j < (DP + 127) / 128; ++j) {
                    constexpr int WORDS = DP == 64 ? 2 : 4;
                    uint32_t x[4][WORDS];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int rr = r + (i & 1) + (i >> 1) * 8;
                        if (DP == 64) {
                            const uint2 u = *(const uint2 *)(v + rr * DP + value_piece<DP>(rr, g >> 1) * 16 + (g & 1) * 8);
                            x[i][0] = u.x, x[i][1] = u.y;
                        } else {
                            const uint4 u = *(const uint4 *)(v + rr * DP + value_piece<DP>(rr, j * 8 + g) * 16);
                            x[i][0] = u.x, x[i][1] = u.y, x[i][WORDS - 2] = u.z, x[i][WORDS - 1] = u.w;
                        }
                    }
#pragma unroll
                    for (int w = 0; w < WORDS; ++w)
#pragma unroll
                        for (int h = 0; h < 2; ++h) { // dims 4 w + 2 h and the next, of this lane's 8 or 16
                            const uint32_t sel = h ? 0x7362 : 0x5140;
                            uint32_t a[4];
                            widen<S8>(prmt(x[0][w], x[1][w], sel), a[0], a[1]);
                            widen<S8>(prmt(x[2][w], x[3][w], sel), a[2], a[3]);
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                mma(o[j * 8 + w * 2 + h][nb], a, pb[nb]);
                                if (FINE) mma(o[j * 8 + w * 2 + h][nb], a, rest[nb]);
                            }
                        }
                }
            }
            __syncwarp(); // the values are read
            if (further < steps_end) copy(VALUES, further, v);
            cp_commit();
            look_up_next(further + WARPS);
            stage = stage + 1 == S::STAGES ? 0 : stage + 1;
        }
        cp_wait<0>();
        __syncwarp();

        // ---- the four warps' parts together
        float *mine = (float *)ring;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const float up[2] = {ex2(k2[nb][0] - P_TOP), ex2(k2[nb][1] - P_TOP)}; // from here on relative to 2^m
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) l[nb][h] += __shfl_xor_sync(~0u, l[nb][h], w);
                // a NaN among the scores, which no maximum shows, is to be the row's result
                if (l[nb][h] != l[nb][h]) m[nb][h] = INFINITY;
                if (g == 0) merge_m[warp][nb * 8 + 2 * t + h] = m[nb][h], merge_l[warp][nb * 8 + 2 * t + h] = l[nb][h];
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                // tile i holds dims d, d + 1 of this lane (as rows g and g + 8 of the instruction)
                const int d = DP == 64 ? g * 8 + i * 2 : (i >> 3) * 128 + g * 16 + (i & 7) * 2;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    *(float2 *)(mine + (nb * 8 + 2 * t + h) * S::PITCH + d) = make_float2(o[i][nb][h] * up[h], o[i][nb][2 + h] * up[h]);
            }
        }
        __syncthreads();
        const bool whole = place_at.whole();
        float *part = parts + place_at.part(blockIdx.x) * part_size;
        const int live = min(rows, ROWS);
        for (int i = tid; i < live * (DP / 4); i += THREADS) {
            const int r = i / (DP / 4), d = (i - r * (DP / 4)) * 4;
            float mm = merge_m[0][r];
#pragma unroll
            for (int w = 1; w < WARPS; ++w) mm = fmaxf(mm, merge_m[w][r]);
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            float ll = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float mw = merge_m[w][r], f = mw == -INFINITY ? 0.f : ex2(mw - mm);
                if (f == 0.f) continue; // nothing seen, or nothing that counts
                const float4 y = *(const float4 *)((const float *)(smem + w * S::RING) + r * S::PITCH + d);
                ll = fmaf(merge_l[w][r], f, ll);
                x.x = fmaf(y.x, f, x.x), x.y = fmaf(y.y, f, x.y), x.z = fmaf(y.z, f, x.z), x.w = fmaf(y.w, f, x.w);
            }
            if (whole) {
                if (d >= c.dim) continue;
                const float inv = ll == 0.f ? 0.f : 1.f / ll;
                const int idx = tile * ROWS + r;
                const int64_t off = (int64_t)(s.begin + idx / group) * p.dst_s0 + (int64_t)(head * group + idx % group) * p.dst_s1 + d;
                *(uint2 *)((char *)p.dst + off * 2) = p.dst_dt == B200_DT_BF16
                        ? make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv))
                        : make_uint2(pack_f16x2(x.x * inv, x.y * inv), pack_f16x2(x.z * inv, x.w * inv));
            } else {
                *(float4 *)(part + 2 * ROWS + r * DP + d) = x;
                if (d == 0) part[r] = mm, part[ROWS + r] = ll;
            }
        }

        // ---- an item in several parts: the last block to finish one puts them together
        if (!whole) {
            const int c0 = place_at.c0, c1 = place_at.c1;
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const bool is_last = atomicAdd(counters + c0, 1u) == (uint32_t)(c1 - c0);
                if (is_last) counters[c0] = 0; // as it was found
                last_part = is_last;
            }
            __syncthreads();
            if (last_part) {
                __threadfence();
                auto part_of = [&](int b) { return parts + place_at.part(b) * part_size; };
                // the parts' weights into shared memory: factor = 2^(m - largest m), then the values eight parts at a time
                const int n = c1 - c0 + 1;
                float *fs = (float *)smem; // [n][ROWS]; the host keeps the grid small enough
                for (int r = warp; r < live; r += WARPS) {
                    float mm = -INFINITY, ll = 0.f;
                    for (int b = lane; b < n; b += 32) {
                        const float mb = __ldcg(part_of(c0 + b) + r);
                        fs[b * ROWS + r] = mb;
                        mm = fmaxf(mm, mb);
                    }
#pragma unroll
                    for (int o = 16; o; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(~0u, mm, o));
                    for (int b = lane; b < n; b += 32) {
                        const float mb = fs[b * ROWS + r], f = mb == -INFINITY ? 0.f : ex2(mb - mm);
                        fs[b * ROWS + r] = f;
                        if (f != 0.f) ll = fmaf(__ldcg(part_of(c0 + b) + ROWS + r), f, ll);
                    }
#pragma unroll
                    for (int o = 16; o; o >>= 1) ll += __shfl_xor_sync(~0u, ll, o);
                    if (lane == 0) merge_l[0][r] = ll;
                }
                __syncthreads();
                for (int i = tid; i < live * (DP / 4); i += THREADS) {
                    const int r = i / (DP / 4), d = (i - r * (DP / 4)) * 4;
                    if (d >= c.dim) continue;
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int base = 0; base < n; base += 8) {
                        float4 y[8];
#pragma unroll
                        for (int u = 0; u < 8; ++u)
                            if (base + u < n) y[u] = __ldcg((const float4 *)(part_of(c0 + base + u) + 2 * ROWS + r * DP + d));
#pragma unroll
                        for (int u = 0; u < 8; ++u) {
                            if (base + u >= n) continue;
                            const float f = fs[(base + u) * ROWS + r];
                            if (f == 0.f) continue;
                            x.x = fmaf(y[u].x, f, x.x), x.y = fmaf(y[u].y, f, x.y), x.z = fmaf(y[u].z, f, x.z), x.w = fmaf(y[u].w, f, x.w);
                        }
                    }
                    const float ll = merge_l[0][r];
                    const float inv = ll == 0.f ? 0.f : 1.f / ll;
                    const int idx = tile * ROWS + r;
                    const int64_t off = (int64_t)(s.begin + idx / group) * p.dst_s0 + (int64_t)(head * group + idx % group) * p.dst_s1 + d;
                    *(uint2 *)((char *)p.dst + off * 2) = p.dst_dt == B200_DT_BF16
                            ? make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv))
                            : make_uint2(pack_f16x2(x.x * inv, x.y * inv), pack_f16x2(x.z * inv, x.w * inv));
                }
            }
        }
        __syncthreads(); // the ring is free for the next item's copies
        if (pieces < CH) {
            // the partial values went over the zeros behind dim
            for (int i = tid; i < WARPS * S::RING / 16; i += THREADS) ((uint4 *)smem)[i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
        }
    }
}

// ---- launch; one file per group of shapes, compiled side by side ------------------------------

template <int DP, int NB, bool S8, bool RUNS, bool FINE>
int run(const b200_kv_attention_params_t &p, int blocks, cudaStream_t cs) {
    using S = shape_t<DP, NB>;
    auto kernel = kv_attention_mma_kernel<DP, NB, S8, RUNS, FINE>;
    // the joining block keeps a factor per part and row in the rings
    const int most = (int)(WARPS * S::RING / (S::ROWS * 4));
    if (blocks > most) blocks = most;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (e != cudaSuccess) return (int)e;
    kernel<<<blocks, THREADS, S::SMEM, cs>>>(p);
    return after_launch();
}
template <int DP, int NB, bool S8, bool RUNS>
int run(const b200_kv_attention_params_t &p, int blocks, cudaStream_t cs) {
    return p.dst_dt == B200_DT_F16 ? run<DP, NB, S8, RUNS, true>(p, blocks, cs) : run<DP, NB, S8, RUNS, false>(p, blocks, cs);
}
template <int DP, int NB>
int run(const b200_kv_attention_params_t &p, int blocks, cudaStream_t cs) {
    // the DP / 16 tokens that a lane copies lie in one page, or may not
    const bool s8 = p.cache.dt == B200_DT_S8;
    if (p.cache.page % (DP / 16) == 0) return s8 ? run<DP, NB, true, true>(p, blocks, cs) : run<DP, NB, false, true>(p, blocks, cs);
    return s8 ? run<DP, NB, true, false>(p, blocks, cs) : run<DP, NB, false, false>(p, blocks, cs);
}

} // namespace kv_mma
} // namespace b200
