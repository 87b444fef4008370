// How the attention kernels divide a ragged batch among the SMs.
//
// An item is one sequence, one key head and ROWS query rows (tokens x the query heads of the key head); it costs its
// tokens, in units of 128, and EXTRA units for what its beginning and end take.  All items side by side -- sequence,
// head, rows -- form one line of units, which is cut into equal parts, one per block, wherever that falls (a part that
// ends within the extra units has no token of that item).  The host knows neither offsets nor lengths, so every
// block derives the line itself, in two short scans over the sequences.
#pragma once

#include "kv_cache.cuh"

namespace b200 {
namespace kv_line {

constexpr int UNIT = 128;
constexpr int LINE_WORDS = 35;

struct item_t {
    int tokens; // that its last row sees
    int units;  // one at least: rows that see nothing are still written
};

// item `tile` of a key head; ones behind the last cost nothing
template <int ROWS>
__device__ __forceinline__ item_t item_of(const seq_t &s, int group, int tile, int64_t capacity) {
    const int rows = (s.end - s.begin) * group;
    item_t i = {0, 0};
    if ((int64_t)tile * ROWS >= rows) return i;
    const int newest = (min((tile + 1) * ROWS, rows) - 1) / group; // the token of its last row
    i.tokens = (int)min((int64_t)max(0, s.first + newest + 1), capacity);
    i.units = max(1, (i.tokens + UNIT - 1) / UNIT);
    return i;
}

// units of one key head of a sequence, the lanes of a warp side by side
template <int ROWS, int EXTRA>
__device__ __forceinline__ int64_t head_units_warp(const seq_t &s, int group, int64_t capacity) {
    const int tiles = ((s.end - s.begin) * group + ROWS - 1) / ROWS;
    int64_t n = 0;
    for (int tile = threadIdx.x & 31; tile < tiles; tile += 32) n += item_of<ROWS>(s, group, tile, capacity).units + EXTRA;
#pragma unroll
    for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(~0u, n, o);
    return n;
}

// the same for a sequence of its own per lane (`there`: the lane has one): short ones by their lanes, the others by the
// whole warp, one after the other
template <int ROWS, int EXTRA>
__device__ __forceinline__ int64_t head_units_lanes(const seq_t &s, bool there, int group, int64_t capacity) {
    const int tiles = there ? ((s.end - s.begin) * group + ROWS - 1) / ROWS : 0;
    int64_t n = 0;
    if (tiles <= 4)
        for (int tile = 0; tile < tiles; ++tile) n += item_of<ROWS>(s, group, tile, capacity).units + EXTRA;
    for (uint32_t todo = __ballot_sync(~0u, tiles > 4); todo; todo &= todo - 1) {
        const int k = __ffs(todo) - 1;
        seq_t one;
        one.begin = __shfl_sync(~0u, s.begin, k);
        one.end = __shfl_sync(~0u, s.end, k);
        one.first = __shfl_sync(~0u, s.first, k);
        const int64_t m = head_units_warp<ROWS, EXTRA>(one, group, capacity);
        if ((int)(threadIdx.x & 31) == k) n = m;
    }
    return n;
}

// inclusive sum over the block's threads (whole warps)
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t *warp_sum) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(~0u, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = v;
    __syncthreads();
    for (int w = 0; w < warp; ++w) v += warp_sum[w];
    return v;
}

// a block's part of the line, and the sequence that it stands in
struct part_t {
    int64_t total, begin, stop;
    int blocks; // that have a part; none is empty
    int group, heads;
    int64_t capacity; // tokens that a row of the table can hold
    int seq;
    int64_t seq_begin, per_head;
    seq_t s;
};

// where a unit lies
struct place_t {
    int head, tile;
    item_t item;
    int64_t item_begin; // on the line
    int u0, u1;         // the item's units of tokens that the block has, none when u1 <= u0
    int64_t next;       // where it goes on
    int c0, c1;         // the blocks that share the item

    __device__ __forceinline__ bool whole() const { return u0 == 0 && u1 == item.units; }
    // a block has two places for partial results: [0] of the item that it begins in, [1] of the one that it ends in
    __device__ __forceinline__ size_t part(int b) const { return (size_t)b * 2 + (b == c0 ? 1 : 0); }
};

// All threads of the block.  False: the block has no part.  `shared`: LINE_WORDS words that nothing else uses meanwhile.
template <int ROWS, int EXTRA, int MIN_PART>
__device__ __forceinline__ bool begin_part(const b200_kv_attention_params_t &p, part_t &l, int64_t *shared) {
    const b200_kv_cache_t &c = p.cache;
    const int tid = threadIdx.x, threads = blockDim.x;
    int64_t *warp_sum = shared, *words = shared + 32;
    l.group = (int)(p.q_heads / c.heads);
    l.heads = (int)c.heads;
    l.capacity = min((int64_t)0x7fffff00, c.table_cols * c.page);
    // the units of `threads` sequences, one per thread, and of all up to this one
    int64_t n = 0, upto = 0;
    auto scan = [&](int base) {
        const int b = base + tid;
        seq_t s = {0, 0, 0};
        if (b < c.seqs) s = load_seq(c, b, p.rows);
        n = head_units_lanes<ROWS, EXTRA>(s, b < c.seqs, l.group, l.capacity) * l.heads;
        upto = block_scan(n, warp_sum);
        if (tid == threads - 1) words[2] = upto;
        if (tid == 0) words[0] = -1;
        __syncthreads();
        return words[2];
    };
    l.total = 0;
    for (int base = 0; base < c.seqs; base += threads) l.total += scan(base);
    // a part has MIN_PART units at least: what it takes to join it is to be less than what it saves
    l.blocks = (int)min((int64_t)gridDim.x, (l.total + MIN_PART - 1) / MIN_PART);
    if (blockIdx.x >= l.blocks) return false;
    l.begin = l.total * blockIdx.x / l.blocks;
    l.stop = l.total * (blockIdx.x + 1) / l.blocks;
    // the sequence that the part begins in, and the units before it
    l.seq_begin = 0;
    for (int base = 0; base < c.seqs; base += threads) {
        int64_t sum = words[2];
        if (c.seqs > threads) { // else the one scan has it
            __syncthreads();
            sum = scan(base);
        }
        if (l.seq_begin + upto > l.begin && l.seq_begin + upto - n <= l.begin) words[0] = base + tid, words[1] = l.seq_begin + upto - n;
        __syncthreads();
        if (words[0] >= 0) break;
        l.seq_begin += sum;
    }
    if (words[0] < 0) return false; // the lengths changed under the kernel
    l.seq = (int)words[0];
    l.seq_begin = words[1];
    l.s = load_seq(c, l.seq, p.rows);
    l.per_head = head_units_warp<ROWS, EXTRA>(l.s, l.group, l.capacity);
    return true;
}

// the block whose part holds unit u
__device__ __forceinline__ int owner(const part_t &l, int64_t u) {
    int64_t o = u * l.blocks / l.total;
    while (l.total * (o + 1) / l.blocks <= u) ++o;
    while (l.total * o / l.blocks > u) --o;
    return (int)o;
}

// what the block has of an item, and who has the rest
template <int EXTRA>
__device__ __forceinline__ void cut(const part_t &l, int64_t at, place_t &q) {
    const int64_t tokens = q.item_begin + EXTRA; // where the item's tokens begin on the line
    q.u0 = (int)max((int64_t)0, at - tokens);
    q.u1 = (int)min((int64_t)q.item.units, l.stop - tokens);
    q.next = tokens + q.item.units;
    q.c0 = owner(l, tokens);
    q.c1 = owner(l, tokens + q.item.units - 1);
}

// the item at unit `at`, which never goes back; whole warps
template <int ROWS, int EXTRA>
__device__ __forceinline__ place_t find_item(const b200_kv_attention_params_t &p, part_t &l, int64_t at) {
    place_t q;
    while (at - l.seq_begin >= l.per_head * l.heads) {
        l.seq_begin += l.per_head * l.heads;
        if (++l.seq >= p.cache.seqs) { // not unless the lengths changed under the kernel
            q.u0 = q.u1 = 0;
            q.next = l.stop;
            return q;
        }
        l.s = load_seq(p.cache, l.seq, p.rows);
        l.per_head = head_units_warp<ROWS, EXTRA>(l.s, l.group, l.capacity);
    }
    q.head = (int)((at - l.seq_begin) / l.per_head);
    q.item_begin = l.seq_begin + q.head * l.per_head;
    const int lane = threadIdx.x & 31;
    q.tile = 0;
    if ((l.s.end - l.s.begin) * l.group <= 4 * ROWS) { // few items: one after the other
        q.item = item_of<ROWS>(l.s, l.group, 0, l.capacity);
        while (at - q.item_begin >= q.item.units + EXTRA) {
            q.item_begin += q.item.units + EXTRA;
            q.item = item_of<ROWS>(l.s, l.group, ++q.tile, l.capacity);
        }
        cut<EXTRA>(l, at, q);
        return q;
    }
    for (;; q.tile += 32) { // 32 items at a time
        const item_t mine = item_of<ROWS>(l.s, l.group, q.tile + lane, l.capacity);
        int64_t upto = mine.units ? mine.units + EXTRA : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t u = __shfl_up_sync(~0u, upto, o);
            if (lane >= o) upto += u;
        }
        const uint32_t here = __ballot_sync(~0u, at - q.item_begin < upto);
        if (here) {
            const int k = __ffs(here) - 1;
            q.tile += k;
            q.item.tokens = __shfl_sync(~0u, mine.tokens, k);
            q.item.units = __shfl_sync(~0u, mine.units, k);
            q.item_begin += __shfl_sync(~0u, upto, k) - q.item.units - EXTRA;
            cut<EXTRA>(l, at, q);
            return q;
        }
        q.item_begin += __shfl_sync(~0u, upto, 31);
    }
}

// Scratch: a counter per block (parts done of the item that begins in its stretch of the line and ends in another's;
// zero between launches), then per block two partial results.
__host__ __device__ inline size_t counter_bytes(int blocks) { return ((size_t)blocks * 4 + 255) / 256 * 256; }

} // namespace kv_line
} // namespace b200
