// Root-mean-square norm of src + residual with the destination quantised on the way
// (b200_rms_norm_launch; the formulas stand with its declaration).
//
// Bound by memory: every element is read once (src, residual) and written once (sum, dst); the row
// stays in registers between the sum of squares and the last product, so the two reductions
// (sum of squares, then the largest |y| that the scale needs) cost no second read.  Per row
// they cost two exchanges among the threads that hold it -- some lanes of a warp for short rows, a block for
// longer ones.  Measured on one B200: 8192 rows of 8192, bf16 with a bf16 residual to e4m3, 82 us (470 MB: 5.7 TB/s, 0.87 of the
// measured copy rate); 262144 rows of 128, bf16 to bf16, 27 us (134 MB: 5.0 TB/s); 1031 rows of 5003, where no
// access can be wider than an element, 25 us (57 MB: 2.3 TB/s).
#include "launch.hpp"
#include "vec8.cuh"

namespace b200 {
namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(~0u, v, o));
    return v;
}

// over all threads of the block (`part`: one word per warp, used once)
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, float *part) {
    v = MAX ? warp_max(v) : warp_sum(v);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) part[warp] = v;
    __syncthreads();
    v = lane < warps ? part[lane] : 0.f; // 0 is neutral for both: magnitudes
    return MAX ? warp_max(v) : warp_sum(v);
}

__device__ __forceinline__ const char *elem(const void *p, int dt, int64_t i) { return (const char *)p + i * (dt_bits(dt) / 8); }

__device__ __forceinline__ bool coded(int dt) { return dt == B200_DT_S8 || dt == B200_DT_F8_E4M3; }

// the VEC elements from c on of a row
template <int VEC>
__device__ __forceinline__ void load_vec(const void *p, int dt, int64_t i, float (&v)[VEC]) {
    if constexpr (VEC == 8) load8(dt, elem(p, dt, i), v);
    else v[0] = load_f32(dt, p, i);
}
// VEC elements of 16 or 32 bits as they are in memory.  The loads of a row are issued with nothing between them, not even
// the look at the type that the conversion needs: with one after the other 8192 rows of 8192 took 160 us.
template <int VEC, bool W32>
struct raw_t;
template <>
struct raw_t<8, false> {
    uint4 u;
    __device__ __forceinline__ void load(const void *p, int64_t i) { u = *(const uint4 *)((const uint16_t *)p + i); }
    __device__ __forceinline__ void get(int dt, float (&v)[8]) const {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = dt == B200_DT_BF16 ? bf16x2_to_f32(w[i]) : f16x2_to_f32(w[i]);
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
    }
};
template <>
struct raw_t<8, true> {
    float4 a, b;
    __device__ __forceinline__ void load(const void *p, int64_t i) {
        a = ((const float4 *)((const float *)p + i))[0];
        b = ((const float4 *)((const float *)p + i))[1];
    }
    __device__ __forceinline__ void get(int, float (&v)[8]) const {
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
};
template <>
struct raw_t<1, false> {
    uint16_t u;
    __device__ __forceinline__ void load(const void *p, int64_t i) { u = ((const uint16_t *)p)[i]; }
    __device__ __forceinline__ void get(int dt, float (&v)[1]) const {
        v[0] = dt == B200_DT_BF16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
    }
};
template <>
struct raw_t<1, true> {
    float a;
    __device__ __forceinline__ void load(const void *p, int64_t i) { a = ((const float *)p)[i]; }
    __device__ __forceinline__ void get(int, float (&v)[1]) const { v[0] = a; }
};
// what the loads have to know: the widths of src and of the residual (none: 0)
enum { W_NONE = 0, W_16 = 1, W_32 = 2 };

template <int VEC>
__device__ __forceinline__ void store_vec(void *p, int dt, int64_t i, const float (&v)[VEC]) {
    if constexpr (VEC == 8) store8(dt, (void *)elem(p, dt, i), v);
    else store1(dt, p, i, v[0]);
}
template <int VEC>
__device__ __forceinline__ void store_codes(const b200_rms_norm_params_t &p, int64_t i, const float (&x)[VEC], float inv) {
    uint8_t *d = (uint8_t *)p.dst + i;
    if constexpr (VEC == 8)
        *(uint2 *)d = make_uint2(codes4(p.dst_dt, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv),
                codes4(p.dst_dt, x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv));
    else *d = code1(p.dst_dt, x[0] * inv);
}

// A block per row: VEC elements per access (8: everything aligned for it; 1: anything), ITER accesses per thread.
template <int VEC, int ITER, int SW, int RW>
__global__ void __launch_bounds__(1024 / (ITER * VEC > 16 ? 2 : 1)) rms_norm_kernel(const __grid_constant__ b200_rms_norm_params_t p) {
    __shared__ float part[2][32];
    const int64_t row = blockIdx.x;
    const int cols = (int)p.cols, step = blockDim.x * VEC, c0 = threadIdx.x * VEC;
    float h[ITER][VEC];
    raw_t<VEC, SW == W_32> s[ITER];
    raw_t<VEC, RW == W_32> r[RW == W_NONE ? 1 : ITER];
#pragma unroll
    for (int i = 0; i < ITER; ++i)
        if (c0 + i * step < cols) s[i].load(p.src, row * p.src_s0 + c0 + i * step);
    if (RW != W_NONE) {
#pragma unroll
        for (int i = 0; i < ITER; ++i)
            if (c0 + i * step < cols) r[RW == W_NONE ? 0 : i].load(p.residual, row * p.residual_s0 + c0 + i * step);
    }
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) h[i][j] = 0.f;
        if (c0 + i * step >= cols) continue;
        s[i].get(p.src_dt, h[i]);
        if (RW != W_NONE) {
            float x[VEC];
            r[RW == W_NONE ? 0 : i].get(p.residual_dt, x);
#pragma unroll
            for (int j = 0; j < VEC; ++j) h[i][j] += x[j];
            store_vec<VEC>(p.sum, p.residual_dt, row * p.sum_s0 + c0 + i * step, h[i]);
        }
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) ss = fmaf(h[i][j], h[i][j], ss);
    ss = row_reduce<false>(ss, part[0]);
    const float rstd = rsqrtf(ss / (float)cols + p.epsilon);
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        // behind the row's end: not even 0 * NaN (of an infinite sum)
        if (c0 + i * step >= cols) continue;
        float g[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[j] = 1.f;
        if (p.gamma) load_vec<VEC>(p.gamma, p.gamma_dt, c0 + i * step, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            h[i][j] = __fmul_rn(__fmul_rn(h[i][j], rstd), g[j]);
            top = max_nan(top, fabsf(h[i][j]));
        }
        if (!coded(p.dst_dt)) store_vec<VEC>(p.dst, p.dst_dt, row * p.dst_s0 + c0 + i * step, h[i]);
    }
    if (!coded(p.dst_dt)) return;
    top = row_reduce<true>(top, part[1]);
    const float scale = max_nan(top * code_peak_factor(p.dst_dt), CODE_SCALE_MIN);
    if (threadIdx.x == 0) p.row_scale[row] = scale;
    const float inv = __frcp_rn(scale);
#pragma unroll
    for (int i = 0; i < ITER; ++i)
        if (c0 + i * step < cols) store_codes<VEC>(p, row * p.dst_s0 + c0 + i * step, h[i], inv);
}

// LANES lanes per row, ITER accesses each, TURNS rows of every group of lanes under way at once; gamma is loaded
// once for them.  Reductions stay inside the group.
template <int VEC, int ITER, int LANES, int TURNS, int SW, int RW>
__global__ void __launch_bounds__(128) rms_norm_short_kernel(const __grid_constant__ b200_rms_norm_params_t p) {
    constexpr int GROUPS = 32 / LANES; // rows side by side in a warp
    const int lane = threadIdx.x & 31, c0 = (lane % LANES) * VEC, cols = (int)p.cols;
    constexpr int step = LANES * VEC;
    const int64_t first = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 5)) * (GROUPS * TURNS) + lane / LANES;
    float h[TURNS][ITER][VEC];
    auto each = [&](auto f) {
#pragma unroll
        for (int k = 0; k < TURNS; ++k)
#pragma unroll
            for (int i = 0; i < ITER; ++i)
                if (first + k * GROUPS < p.rows && c0 + i * step < cols) f(first + k * GROUPS, c0 + i * step, h[k][i]);
    };
#pragma unroll
    for (int k = 0; k < TURNS; ++k)
#pragma unroll
        for (int i = 0; i < ITER; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) h[k][i][j] = 0.f;
    raw_t<VEC, SW == W_32> s[TURNS][ITER];
    raw_t<VEC, RW == W_32> r[TURNS][ITER];
#pragma unroll
    for (int k = 0; k < TURNS; ++k)
#pragma unroll
        for (int i = 0; i < ITER; ++i)
            if (first + k * GROUPS < p.rows && c0 + i * step < cols) {
                s[k][i].load(p.src, (first + k * GROUPS) * p.src_s0 + c0 + i * step);
                if (RW != W_NONE) r[k][i].load(p.residual, (first + k * GROUPS) * p.residual_s0 + c0 + i * step);
            }
#pragma unroll
    for (int k = 0; k < TURNS; ++k)
#pragma unroll
        for (int i = 0; i < ITER; ++i)
            if (first + k * GROUPS < p.rows && c0 + i * step < cols) {
                s[k][i].get(p.src_dt, h[k][i]);
                if (RW != W_NONE) {
                    float x[VEC];
                    r[k][i].get(p.residual_dt, x);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) h[k][i][j] += x[j];
                    store_vec<VEC>(p.sum, p.residual_dt, (first + k * GROUPS) * p.sum_s0 + c0 + i * step, h[k][i]);
                }
            }
    float rstd[TURNS], top[TURNS];
#pragma unroll
    for (int k = 0; k < TURNS; ++k) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < ITER; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) ss = fmaf(h[k][i][j], h[k][i][j], ss);
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
        rstd[k] = rsqrtf(ss / (float)cols + p.epsilon);
        top[k] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        if (c0 + i * step >= cols) continue;
        float g[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[j] = 1.f;
        if (p.gamma) load_vec<VEC>(p.gamma, p.gamma_dt, c0 + i * step, g);
#pragma unroll
        for (int k = 0; k < TURNS; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                h[k][i][j] = __fmul_rn(__fmul_rn(h[k][i][j], rstd[k]), g[j]);
                top[k] = max_nan(top[k], fabsf(h[k][i][j]));
            }
    }
    if (!coded(p.dst_dt)) {
        each([&](int64_t row, int c, float(&v)[VEC]) { store_vec<VEC>(p.dst, p.dst_dt, row * p.dst_s0 + c, v); });
        return;
    }
#pragma unroll
    for (int k = 0; k < TURNS; ++k) {
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1) top[k] = max_nan(top[k], __shfl_xor_sync(~0u, top[k], o));
        const int64_t row = first + k * GROUPS;
        if (row >= p.rows) continue;
        const float scale = max_nan(top[k] * code_peak_factor(p.dst_dt), CODE_SCALE_MIN);
        if (lane % LANES == 0) p.row_scale[row] = scale;
        const float inv = __frcp_rn(scale);
#pragma unroll
        for (int i = 0; i < ITER; ++i)
            if (c0 + i * step < cols) store_codes<VEC>(p, row * p.dst_s0 + c0 + i * step, h[k][i], inv);
    }
}

// rows longer than the registers of a block: src and residual are read once per pass (three for an
// 8-bit destination), from L2 after the first
__global__ void __launch_bounds__(1024) rms_norm_long_kernel(const __grid_constant__ b200_rms_norm_params_t p) {
    __shared__ float part[2][32];
    const int64_t row = blockIdx.x;
    auto value = [&](int64_t c) {
        float v = load_f32(p.src_dt, p.src, row * p.src_s0 + c);
        return p.residual ? v + load_f32(p.residual_dt, p.residual, row * p.residual_s0 + c) : v;
    };
    float ss = 0.f;
    for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) {
        const float v = value(c);
        ss = fmaf(v, v, ss);
    }
    ss = row_reduce<false>(ss, part[0]);
    const float rstd = rsqrtf(ss / (float)p.cols + p.epsilon);
    auto normed = [&](float v, int64_t c) {
        return __fmul_rn(__fmul_rn(v, rstd), p.gamma ? load_f32(p.gamma_dt, p.gamma, c) : 1.f);
    };
    float inv = 0.f;
    if (coded(p.dst_dt)) {
        float top = 0.f;
        for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) top = max_nan(top, fabsf(normed(value(c), c)));
        top = row_reduce<true>(top, part[1]);
        const float scale = max_nan(top * code_peak_factor(p.dst_dt), CODE_SCALE_MIN);
        if (threadIdx.x == 0) p.row_scale[row] = scale;
        inv = __frcp_rn(scale);
    }
    // sum may be the residual's or src's own memory: each element is read here before it is written
    for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) {
        const float v = value(c), y = normed(v, c);
        if (p.residual) store1(p.residual_dt, p.sum, row * p.sum_s0 + c, v);
        if (coded(p.dst_dt)) ((uint8_t *)p.dst)[row * p.dst_s0 + c] = code1(p.dst_dt, y * inv);
        else store1(p.dst_dt, p.dst, row * p.dst_s0 + c, y);
    }
}

bool aligned_rows(const void *p, int dt, int64_t s0) {
    return !p || (((uintptr_t)p | (uintptr_t)(s0 * (dt_bits(dt) / 8))) % (dt_bits(dt) == 8 ? 8 : 16)) == 0;
}

template <int VEC, int ITER, int SW, int RW>
int run(const b200_rms_norm_params_t &p, cudaStream_t cs) {
    const int64_t per = (int64_t)VEC * ITER * 32;
    rms_norm_kernel<VEC, ITER, SW, RW><<<(unsigned)p.rows, (unsigned)((p.cols + per - 1) / per) * 32, 0, cs>>>(p);
    return after_launch();
}
template <int VEC, int ITER, int LANES, int TURNS, int SW, int RW>
int run_short(const b200_rms_norm_params_t &p, cudaStream_t cs) {
    const int64_t per = 4 * (32 / LANES) * TURNS; // rows of a block
    rms_norm_short_kernel<VEC, ITER, LANES, TURNS, SW, RW><<<(unsigned)((p.rows + per - 1) / per), 128, 0, cs>>>(p);
    return after_launch();
}

template <int SW, int RW>
int choose(const b200_rms_norm_params_t &p, bool vec, cudaStream_t cs) {
    // Few rows: as many threads as the row has accesses, the row's latency is what counts.  Many: four accesses per
    // thread, whose instructions and reductions then cost a third.
    const bool few = p.rows <= 256;
    if (vec) {
        if (p.cols <= 64) return run_short<8, 1, 8, 4, SW, RW>(p, cs);
        if (p.cols <= 128) return run_short<8, 1, 16, 4, SW, RW>(p, cs);
        if (p.cols <= 256) return run_short<8, 1, 32, 4, SW, RW>(p, cs);
        if (p.cols <= 1024 && !few) return run_short<8, 4, 32, 1, SW, RW>(p, cs);
        if (p.cols <= 8 * 1024 && few) return run<8, 1, SW, RW>(p, cs);
        if (p.cols <= 16 * 1024) return run<8, 4, SW, RW>(p, cs);
    } else {
        if (p.cols <= 256) return run_short<1, 8, 32, 1, SW, RW>(p, cs);
        if (p.cols <= 8 * 1024) return run<1, 8, SW, RW>(p, cs);
        if (p.cols <= 16 * 1024) return run<1, 32, SW, RW>(p, cs);
    }
    rms_norm_long_kernel<<<(unsigned)p.rows, 1024, 0, cs>>>(p);
    return after_launch();
}

bool is_f(int dt) { return dt == B200_DT_F32 || dt == B200_DT_BF16 || dt == B200_DT_F16; }

} // namespace
} // namespace b200

using namespace b200;

extern "C" B200_API int b200_rms_norm_launch(const b200_rms_norm_params_t *pp, b200_stream_t stream) {
    if (!pp) return B200_ERR_BAD_ARG;
    const b200_rms_norm_params_t &p = *pp;
    const bool coded = p.dst_dt == B200_DT_S8 || p.dst_dt == B200_DT_F8_E4M3;
    if (!is_f(p.src_dt) || (!is_f(p.dst_dt) && !coded)) return B200_ERR_UNSUPPORTED;
    if ((p.residual && !is_f(p.residual_dt)) || (p.gamma && !is_f(p.gamma_dt))) return B200_ERR_UNSUPPORTED;
    if (p.rows < 0 || p.cols < 0 || p.rows > 0x7fffffff || p.cols > 0x7fffffff) return B200_ERR_BAD_ARG;
    if (p.rows == 0 || p.cols == 0) return 0;
    if (!p.src || !p.dst || (p.residual && !p.sum) || (coded && !p.row_scale)) return B200_ERR_BAD_ARG;
    cudaStream_t cs = (cudaStream_t)stream;
    const bool vec = p.cols % 8 == 0 && aligned_rows(p.src, p.src_dt, p.src_s0) && aligned_rows(p.residual, p.residual_dt, p.residual_s0)
            && aligned_rows(p.residual ? p.sum : nullptr, p.residual_dt, p.sum_s0) && aligned_rows(p.gamma, p.gamma_dt, 0)
            && aligned_rows(p.dst, p.dst_dt, p.dst_s0);
    const bool s32 = p.src_dt == B200_DT_F32;
    if (!p.residual) return s32 ? choose<W_32, W_NONE>(p, vec, cs) : choose<W_16, W_NONE>(p, vec, cs);
    if (p.residual_dt == B200_DT_F32) return s32 ? choose<W_32, W_32>(p, vec, cs) : choose<W_16, W_32>(p, vec, cs);
    return s32 ? choose<W_32, W_16>(p, vec, cs) : choose<W_16, W_16>(p, vec, cs);
}
