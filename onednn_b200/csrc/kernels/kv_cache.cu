// The paged 8-bit cache of keys and values: quantising new tokens into it (b200_kv_append_launch) and
// reading tokens back (b200_kv_read_launch).  The arithmetic stands with the declarations.
//
// Both move each byte once: new rows stay in registers between finding their page's scale and rounding.  Measured on one B200,
// 8 heads of 128, bf16 rows, s8: 10287 new tokens appended in 27 us (63 MB: 2.3 TB/s; rounding and packing take
// two thirds of the issue slots), 16152 read in 24 us (99 MB: 4.1 TB/s).  A step of one token per sequence takes 7 us each:
// the launch, then where a row's sequence, its page and its scale are, one load behind the other.
#include "kv_cache.cuh"
#include "launch.hpp"

namespace b200 {
namespace {

constexpr int APPEND_THREADS = 128;

__device__ __forceinline__ float finite_abs(float x) {
    x = fabsf(x);
    return x < __int_as_float(0x7f800000) ? x : 0.f; // neither infinity nor NaN
}
__device__ __forceinline__ float no_nan(float x) { return x == x ? x : 0.f; }

// magnitudes' bits of eight 16-bit values against the largest so far, even and odd elements side by side
__device__ __forceinline__ uint32_t top_bits(uint32_t top, const uint4 &u) {
    return __vmaxu2(__vmaxu2(top, u.x & 0x7fff7fffu), __vmaxu2(__vmaxu2(u.y & 0x7fff7fffu, u.z & 0x7fff7fffu), u.w & 0x7fff7fffu));
}
__device__ __forceinline__ void widen8(bool bf16, const uint4 &u, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = bf16 ? bf16x2_to_f32(w[i]) : f16x2_to_f32(w[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}

// The new tokens of one sequence in one page, one head: the largest magnitude, the page's scale,
// the codes.  All threads of the block, and no two blocks on the same page and head.
template <bool VEC>
__device__ __forceinline__ void append_page(const b200_kv_rows_params_t &p, const char *src, uint8_t *codes, float *scale_at,
        int64_t row, int slot, int count, float *part) {
    const b200_kv_cache_t &c = p.cache;
    const int dim = (int)c.dim, tid = threadIdx.x;
    const int unit = VEC ? 8 : 1, per = dim / unit, esize = dt_bits(p.dt) / 8;
    const char *rows = src + row * p.s_row * esize;
    float top = 0.f;
    // 16-bit rows of up to KEEP accesses per thread stay in registers between the two passes, as long as all values are finite
    constexpr int KEEP = VEC ? 8 : 1;
    uint4 kept[KEEP];
    bool keep = VEC && p.dt != B200_DT_F32 && count * per <= KEEP * APPEND_THREADS;
    const bool bf16 = p.dt == B200_DT_BF16;
    if (keep) {
        uint32_t bits = 0;
#pragma unroll
        for (int k = 0; k < KEEP; ++k) {
            const int i = k * APPEND_THREADS + tid, r = i / per;
            kept[k] = make_uint4(0, 0, 0, 0);
            if (i < count * per) kept[k] = *(const uint4 *)(rows + (r * p.s_row + (i - r * per) * 8) * 2);
        }
#pragma unroll
        for (int k = 0; k < KEEP; ++k) bits = top_bits(bits, kept[k]);
        const float2 f = bf16 ? bf16x2_to_f32(bits) : f16x2_to_f32(bits);
        top = fmaxf(f.x, f.y);
        keep = !__syncthreads_or(!(f.x < INFINITY && f.y < INFINITY)); // an infinity or NaN does not count: value by value, below
        if (!keep) top = 0.f;
    }
    for (int i = keep ? count * per : tid; i < count * per; i += APPEND_THREADS) {
        const int r = i / per, e = (i - r * per) * unit;
        const char *at = rows + (r * p.s_row + e) * esize;
        if (VEC) {
            float v[8];
            load8(p.dt, at, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, finite_abs(v[j]));
        } else {
            top = fmaxf(top, finite_abs(load_f32(p.dt, at, 0)));
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    if ((tid & 31) == 0) part[tid >> 5] = top;
    const float old = slot > 0 ? *scale_at : 0.f;
    __syncthreads(); // all have read the old scale
    top = part[0];
#pragma unroll
    for (int w = 1; w < APPEND_THREADS / 32; ++w) top = fmaxf(top, part[w]);
    const float scale = fmaxf(fmaxf(top * code_peak_factor(c.dt), CODE_SCALE_MIN), old);
    const float inv = __frcp_rn(scale);
    if (tid == 0) *scale_at = scale;
    if (slot > 0 && scale > old) {
        const float factor = __fdiv_rn(old, scale);
        for (int i = tid; i < slot * per; i += APPEND_THREADS) {
            const int r = i / per, e = (i - r * per) * unit;
            uint8_t *at = codes + r * c.s_slot + e;
            if (VEC) {
                const uint2 w = *(const uint2 *)at;
                float a[4], b[4];
                code_values4(c.dt, w.x, a);
                code_values4(c.dt, w.y, b);
                *(uint2 *)at = make_uint2(codes4(c.dt, a[0] * factor, a[1] * factor, a[2] * factor, a[3] * factor),
                        codes4(c.dt, b[0] * factor, b[1] * factor, b[2] * factor, b[3] * factor));
            } else {
                *at = code1(c.dt, code_value(c.dt, *at) * factor);
            }
        }
    }
    codes += (int64_t)slot * c.s_slot;
    if (keep) {
#pragma unroll
        for (int k = 0; k < KEEP; ++k) {
            const int i = k * APPEND_THREADS + tid, r = i / per;
            if (i >= count * per) break;
            float v[8];
            widen8(bf16, kept[k], v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= inv;
            *(uint2 *)(codes + r * c.s_slot + (i - r * per) * 8) = make_uint2(codes4(c.dt, v[0], v[1], v[2], v[3]), codes4(c.dt, v[4], v[5], v[6], v[7]));
        }
    }
    for (int i = keep ? count * per : tid; i < count * per; i += APPEND_THREADS) {
        const int r = i / per, e = (i - r * per) * unit;
        const char *at = rows + (r * p.s_row + e) * esize;
        uint8_t *d = codes + r * c.s_slot + e;
        if (VEC) {
            float v[8];
            load8(p.dt, at, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = held(c.dt, no_nan(v[j]) * inv);
            *(uint2 *)d = make_uint2(codes4(c.dt, v[0], v[1], v[2], v[3]), codes4(c.dt, v[4], v[5], v[6], v[7]));
        } else {
            *d = code1(c.dt, held(c.dt, no_nan(load_f32(p.dt, at, 0)) * inv));
        }
    }
    __syncthreads(); // `part` is free again
}

// Block (x, head, key or value) owns the pages whose first new token is one of `span` rows.  The host
// does not know where sequences begin, so every block looks: the threads compare one
// sequence each with its row.
template <bool VEC>
__global__ void __launch_bounds__(APPEND_THREADS) kv_append_kernel(const __grid_constant__ b200_kv_rows_params_t p, int span) {
    __shared__ float part[APPEND_THREADS / 32];
    __shared__ int found;
    const b200_kv_cache_t &c = p.cache;
    const int head = blockIdx.y, page = (int)c.page, tid = threadIdx.x;
    const char *src = (const char *)(blockIdx.z ? p.value : p.key) + head * p.s_head * (dt_bits(p.dt) / 8);
    uint8_t *base = (uint8_t *)(blockIdx.z ? c.value : c.key) + head * c.s_head;
    float *scales = (blockIdx.z ? c.value_scale : c.key_scale) + head;
    int64_t row = (int64_t)blockIdx.x * span;
    const int64_t stop = min(row + span, p.rows);
    while (row < stop) {
        // the sequence that the row belongs to, or else the next one that has rows
        if (tid == 0) found = 0x7fffffff;
        __syncthreads();
        for (int b = tid; b < c.seqs; b += APPEND_THREADS) {
            const int hi = c.offsets[b + 1];
            if (hi > row && hi > c.offsets[b]) {
                atomicMin(&found, b);
                break;
            }
        }
        __syncthreads();
        const int b = found;
        __syncthreads(); // read before it is set again
        if (b == 0x7fffffff) return;
        const seq_t s = load_seq(c, b, p.rows);
        // the first row at or behind `row` that is the first new one of a page
        int64_t lead = max(row, (int64_t)s.begin - min(s.first, 0));
        const int64_t start = s.begin - min(s.first, 0); // of token 0 or `first`
        if (lead > start) {
            const int at = s.first + (int)(lead - s.begin), slot = at % page;
            if (slot) lead += page - slot;
        }
        if (lead >= s.end) { // no page of this sequence begins here any more
            row = max((int64_t)s.end, row + 1);
            continue;
        }
        if (lead >= stop) return;
        const int at = s.first + (int)(lead - s.begin);
        int slot;
        const int phys = page_of(c, b, at, slot);
        const int count = (int)min((int64_t)page - slot, s.end - lead);
        if (phys < 0) {
            if (tid == 0) flag_bad_page(c);
        } else {
            append_page<VEC>(p, src, base + phys * c.s_page, scales + (int64_t)phys * c.heads, lead, slot, count, part);
        }
        row = lead + count;
    }
}

template <bool VEC>
__device__ __forceinline__ void read_row(const b200_kv_rows_params_t &p, const seq_t &s, int b, int64_t row, int lane) {
    const b200_kv_cache_t &c = p.cache;
    const int at = s.first + (int)(row - s.begin);
    int slot = 0, phys = -1;
    if (at >= 0) {
        phys = page_of(c, b, at, slot);
        if (phys < 0 && lane == 0) flag_bad_page(c);
    }
    const int unit = VEC ? 16 : 1, esize = dt_bits(p.dt) / 8;
    const uint32_t per = (uint32_t)c.dim / unit, all = per * (uint32_t)c.heads; // 2^30 at most: twice that, and the step behind it, fit
    const int64_t place = (int64_t)phys * c.s_page + (int64_t)slot * c.s_slot;
    auto put = [&](char *d, const uint4 &w, float scale) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float a[4], bb[4], v[8];
            code_values4(c.dt, u[2 * j], a);
            code_values4(c.dt, u[2 * j + 1], bb);
#pragma unroll
            for (int t = 0; t < 4; ++t) v[t] = a[t] * scale, v[4 + t] = bb[t] * scale;
            store8(p.dt, d + 8 * j * esize, v);
        }
    };
    for (uint32_t i = lane; i < 2 * all; i += 32) {
        const bool val = i >= all;
        const uint32_t k = val ? i - all : i, head = k / per, e = (k - head * per) * unit;
        char *d = (char *)(val ? p.value : p.key) + (row * p.s_row + head * p.s_head + e) * esize;
        const uint8_t *from = (const uint8_t *)(val ? c.value : c.key) + place + head * c.s_head + e;
        const float scale = phys < 0 ? 0.f : (val ? c.value_scale : c.key_scale)[(int64_t)phys * c.heads + head];
        if (VEC) put(d, phys < 0 ? make_uint4(0, 0, 0, 0) : *(const uint4 *)from, scale);
        else store1(p.dt, d, 0, phys < 0 ? 0.f : code_value(c.dt, *from) * scale);
    }
}

// One warp per row: keys and values of all heads of one token.
template <bool VEC>
__global__ void __launch_bounds__(128) kv_read_kernel(const __grid_constant__ b200_kv_rows_params_t p) {
    const b200_kv_cache_t &c = p.cache;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= p.rows) return;
    for (int base = 0; base < c.seqs; base += 32) {
        const int i = base + lane;
        const bool in = i < c.seqs && c.offsets[i] <= row && row < c.offsets[i + 1];
        const uint32_t m = __ballot_sync(~0u, in);
        if (m) {
            const int b = base + __ffs(m) - 1;
            read_row<VEC>(p, load_seq(c, b, p.rows), b, row, lane);
            return;
        }
    }
}

int check(const b200_kv_rows_params_t *p) {
    if (!p) return B200_ERR_BAD_ARG;
    if (!kv_cache_ok(p->cache) || p->rows < 0 || p->rows > 0x7fffffff) return B200_ERR_BAD_ARG;
    if (p->dt != B200_DT_F32 && p->dt != B200_DT_BF16 && p->dt != B200_DT_F16) return B200_ERR_UNSUPPORTED;
    if (p->rows > 0 && p->cache.seqs > 0 && (!p->key || !p->value)) return B200_ERR_BAD_ARG;
    return 0;
}

// `unit` elements of dim at a time: rows, heads and pages all start where such an access may
bool vector_ok(const b200_kv_rows_params_t &p, int unit) {
    const b200_kv_cache_t &c = p.cache;
    const int esize = dt_bits(p.dt) / 8;
    const uintptr_t rows = (uintptr_t)p.key | (uintptr_t)p.value | (uintptr_t)(p.s_row * esize) | (uintptr_t)(p.s_head * esize);
    const uintptr_t codes = (uintptr_t)c.key | (uintptr_t)c.value | (uintptr_t)c.s_page | (uintptr_t)c.s_head | (uintptr_t)c.s_slot;
    return c.dim % unit == 0 && rows % 16 == 0 && codes % unit == 0;
}

} // namespace
} // namespace b200

using namespace b200;

extern "C" B200_API int b200_kv_append_launch(const b200_kv_rows_params_t *p, b200_stream_t stream) {
    const int rc = check(p);
    if (rc) return rc;
    if (p->rows == 0 || p->cache.seqs == 0) return 0;
    // A block looks through as many rows as a sequence has on average, at most a page of them: one
    // row where every sequence brings one token, so that all pages are written side by side.
    const int64_t mean = p->rows / p->cache.seqs;
    const int span = (int)(mean < 1 ? 1 : mean < p->cache.page ? mean : p->cache.page);
    const dim3 grid((unsigned)((p->rows + span - 1) / span), (unsigned)p->cache.heads, 2);
    if (vector_ok(*p, 8)) kv_append_kernel<true><<<grid, APPEND_THREADS, 0, (cudaStream_t)stream>>>(*p, span);
    else kv_append_kernel<false><<<grid, APPEND_THREADS, 0, (cudaStream_t)stream>>>(*p, span);
    return after_launch();
}

extern "C" B200_API int b200_kv_read_launch(const b200_kv_rows_params_t *p, b200_stream_t stream) {
    const int rc = check(p);
    if (rc) return rc;
    if (p->rows == 0 || p->cache.seqs == 0) return 0;
    const unsigned grid = (unsigned)((p->rows + 3) / 4);
    if (vector_ok(*p, 16)) kv_read_kernel<true><<<grid, 128, 0, (cudaStream_t)stream>>>(*p);
    else kv_read_kernel<false><<<grid, 128, 0, (cudaStream_t)stream>>>(*p);
    return after_launch();
}
