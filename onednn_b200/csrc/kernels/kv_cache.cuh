// The paged cache and the ragged batch over it, as every kernel that touches them sees them.
// Offsets, lengths and page indices are data of the caller: nothing here follows one that
// would leave its tensor.
#pragma once

#include "vec8.cuh"

namespace b200 {

// rows of sequence b, held inside the tensor's `rows`
struct seq_t {
    int begin, end; // rows
    int first;      // the token that row `begin` stands for; below zero when there are more rows than tokens
};

__device__ __forceinline__ seq_t load_seq(const b200_kv_cache_t &c, int b, int64_t rows) {
    seq_t s;
    const int lo = c.offsets[b], hi = c.offsets[b + 1], len = c.lens[b];
    s.begin = min(max(lo, 0), (int)rows);
    s.end = max(s.begin, min(hi, (int)rows));
    // len - n may leave 32 bits only for lengths that no table holds
    const int64_t first = (int64_t)max(len, 0) - ((int64_t)hi - lo) + (s.begin - lo);
    s.first = (int)(first < -0x40000000 ? -0x40000000 : first);
    return s;
}

// the page that holds token `at` (>= 0), or -1: beyond the table, or an index outside the cache
__device__ __forceinline__ int page_of(const b200_kv_cache_t &c, int b, int at, int &slot) {
    const int j = at / (int)c.page;
    slot = at - j * (int)c.page;
    if (j >= c.table_cols) return -1;
    const int page = c.table[(int64_t)b * c.table_s0 + j];
    return (page >= 0 && page < c.pages) ? page : -1;
}

__device__ __forceinline__ void flag_bad_page(const b200_kv_cache_t &c) {
    if (c.status) atomicOr(c.status, B200_STATUS_BAD_PAGE);
}

inline bool kv_cache_ok(const b200_kv_cache_t &c) {
    if (c.dt != B200_DT_S8 && c.dt != B200_DT_F8_E4M3) return false;
    if (c.pages < 0 || c.pages > 0x7fffffff || c.heads < 1 || c.heads > 65535 || c.page < 1 || c.page > (1 << 20) || c.dim < 1)
        return false;
    if (c.dim > (1 << 20) || c.page * c.dim > (1 << 30) || c.heads * c.dim > (1 << 30)) return false; // counted in 32 bits
    if (c.seqs < 0 || c.seqs > (1 << 24) || c.table_cols < 0) return false;
    if (c.seqs > 0 && (!c.offsets || !c.lens || (c.table_cols > 0 && !c.table))) return false;
    return c.pages == 0 || (c.key && c.value && c.key_scale && c.value_scale);
}

} // namespace b200
