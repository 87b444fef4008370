// Root-mean-square norm of src + residual with the destination quantised on the way
// (b200_rms_norm_launch; the formulas stand with its declaration).
//
// Bound by memory: every element is read once (src, residual) and written once (sum, dst); the row
// stays in registers between the sum of squares and the last product, so the two reductions
// (sum of squares, then the largest |y| that the scale needs) cost no second read.  Per row
// they cost two exchanges among the threads that hold it -- one warp for short rows, a block for
// longer ones.
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

// over all threads of the row: a warp, or the block (`part`: one word per warp, used once per call)
template <bool WARP, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float *part) {
    v = MAX ? warp_max(v) : warp_sum(v);
    if (WARP) return v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) part[warp] = v;
    __syncthreads();
    v = lane < warps ? part[lane] : 0.f; // 0 is neutral for both: magnitudes
    return MAX ? warp_max(v) : warp_sum(v);
}

__device__ __forceinline__ const char *elem(const void *p, int dt, int64_t i) { return (const char *)p + i * (dt_bits(dt) / 8); }

// VEC elements per access (8: everything aligned for it; 1: anything), ITER accesses per thread and
// row.  WARP: one warp per row, else one block per row.
template <int VEC, int ITER, bool WARP>
__global__ void __launch_bounds__(1024) rms_norm_kernel(const __grid_constant__ b200_rms_norm_params_t p) {
    __shared__ float part[2][32];
    const int lanes = WARP ? 32 : blockDim.x, lane = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int64_t row = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    if (WARP && row >= p.rows) return;
    const int cols = (int)p.cols;
    float h[ITER][VEC];
    // all loads of the row first
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int c = (i * lanes + lane) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) h[i][j] = 0.f;
        if (c < cols) {
            if constexpr (VEC == 8) load8(p.src_dt, elem(p.src, p.src_dt, row * p.src_s0 + c), h[i]);
            else h[i][0] = load_f32(p.src_dt, p.src, row * p.src_s0 + c);
        }
    }
    if (p.residual) {
        float r[ITER][VEC];
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (i * lanes + lane) * VEC;
#pragma unroll
            for (int j = 0; j < VEC; ++j) r[i][j] = 0.f;
            if (c < cols) {
                if constexpr (VEC == 8) load8(p.residual_dt, elem(p.residual, p.residual_dt, row * p.residual_s0 + c), r[i]);
                else r[i][0] = load_f32(p.residual_dt, p.residual, row * p.residual_s0 + c);
            }
        }
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (i * lanes + lane) * VEC;
#pragma unroll
            for (int j = 0; j < VEC; ++j) h[i][j] += r[i][j];
            if (c < cols) {
                if constexpr (VEC == 8) store8(p.residual_dt, (void *)elem(p.sum, p.residual_dt, row * p.sum_s0 + c), h[i]);
                else store1(p.residual_dt, p.sum, row * p.sum_s0 + c, h[i][0]);
            }
        }
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) ss = fmaf(h[i][j], h[i][j], ss);
    ss = row_reduce<WARP, false>(ss, part[0]);
    const float rstd = rsqrtf(ss / (float)cols + p.epsilon);
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int c = (i * lanes + lane) * VEC;
        float g[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[j] = 1.f;
        if (p.gamma && c < cols) {
            if constexpr (VEC == 8) load8(p.gamma_dt, elem(p.gamma, p.gamma_dt, c), g);
            else g[0] = load_f32(p.gamma_dt, p.gamma, c);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            h[i][j] = __fmul_rn(__fmul_rn(h[i][j], rstd), g[j]);
            // threads behind the row's end hold zeros, which 0 * NaN (an infinite sum) would spoil
            if (VEC == 8 || c < cols) top = max_nan(top, c < cols ? fabsf(h[i][j]) : 0.f);
        }
    }
    if (p.dst_dt == B200_DT_S8 || p.dst_dt == B200_DT_F8_E4M3) {
        top = row_reduce<WARP, true>(top, part[1]);
        const float scale = max_nan(top * code_peak_factor(p.dst_dt), CODE_SCALE_MIN);
        if (lane == 0) p.row_scale[row] = scale;
        const float inv = __frcp_rn(scale);
        uint8_t *d = (uint8_t *)p.dst + row * p.dst_s0;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (i * lanes + lane) * VEC;
            if (c >= cols) continue;
            if constexpr (VEC == 8) {
                float *x = h[i];
                *(uint2 *)(d + c) = make_uint2(codes4(p.dst_dt, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv),
                        codes4(p.dst_dt, x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv));
            } else {
                d[c] = code1(p.dst_dt, h[i][0] * inv);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (i * lanes + lane) * VEC;
            if (c >= cols) continue;
            if constexpr (VEC == 8) store8(p.dst_dt, (void *)elem(p.dst, p.dst_dt, row * p.dst_s0 + c), h[i]);
            else store1(p.dst_dt, p.dst, row * p.dst_s0 + c, h[i][0]);
        }
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
    ss = row_reduce<false, false>(ss, part[0]);
    const float rstd = rsqrtf(ss / (float)p.cols + p.epsilon);
    auto normed = [&](float v, int64_t c) {
        return __fmul_rn(__fmul_rn(v, rstd), p.gamma ? load_f32(p.gamma_dt, p.gamma, c) : 1.f);
    };
    const bool coded = p.dst_dt == B200_DT_S8 || p.dst_dt == B200_DT_F8_E4M3;
    float inv = 0.f;
    if (coded) {
        float top = 0.f;
        for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) top = max_nan(top, fabsf(normed(value(c), c)));
        top = row_reduce<false, true>(top, part[1]);
        const float scale = max_nan(top * code_peak_factor(p.dst_dt), CODE_SCALE_MIN);
        if (threadIdx.x == 0) p.row_scale[row] = scale;
        inv = __frcp_rn(scale);
    }
    // sum may be the residual's or src's own memory: each element is read here before it is written
    for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) {
        const float v = value(c), y = normed(v, c);
        if (p.residual) store1(p.residual_dt, p.sum, row * p.sum_s0 + c, v);
        if (coded) ((uint8_t *)p.dst)[row * p.dst_s0 + c] = code1(p.dst_dt, y * inv);
        else store1(p.dst_dt, p.dst, row * p.dst_s0 + c, y);
    }
}

bool aligned_rows(const void *p, int dt, int64_t s0) {
    return !p || (((uintptr_t)p | (uintptr_t)(s0 * (dt_bits(dt) / 8))) % (dt_bits(dt) == 8 ? 8 : 16)) == 0;
}

template <int VEC, int ITER, bool WARP>
int run(const b200_rms_norm_params_t &p, cudaStream_t cs) {
    if (WARP) {
        // four rows per block: enough blocks to spread few rows, enough warps for many
        const int64_t blocks = (p.rows + 3) / 4;
        rms_norm_kernel<VEC, ITER, true><<<(unsigned)blocks, 128, 0, cs>>>(p);
    } else {
        const int64_t per = (int64_t)VEC * ITER * 32;
        const int threads = (int)((p.cols + per - 1) / per) * 32;
        rms_norm_kernel<VEC, ITER, false><<<(unsigned)p.rows, threads, 0, cs>>>(p);
    }
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
    if (vec) {
        if (p.cols <= 256) return run<8, 1, true>(p, cs);
        if (p.cols <= 1024) return run<8, 4, true>(p, cs);
        if (p.cols <= 8 * 1024) return run<8, 1, false>(p, cs);
        if (p.cols <= 32 * 1024) return run<8, 4, false>(p, cs);
    } else {
        if (p.cols <= 256) return run<1, 8, true>(p, cs);
        if (p.cols <= 8 * 1024) return run<1, 8, false>(p, cs);
        if (p.cols <= 32 * 1024) return run<1, 32, false>(p, cs);
    }
    rms_norm_long_kernel<<<(unsigned)p.rows, 1024, 0, cs>>>(p);
    return after_launch();
}
