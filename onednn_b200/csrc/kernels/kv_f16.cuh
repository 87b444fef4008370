// Codes and weights as f16 operands of the attention kernels' products, and what both kernels say in PTX.
#pragma once

#include "kv_cache.cuh"

namespace b200 {

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float min_nan(float a, float b) { // keeps a NaN
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint16_t v) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
    return r;
}
// four codes -> two f16 pairs, exactly.  s8: code + 128 in the low byte of 0x6400 (1024), minus 1152.
template <bool S8>
__device__ __forceinline__ void widen(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if (S8) {
        w ^= 0x80808080u;
        lo = hsub2(__byte_perm(w, 0x64646464u, 0x4140), 0x64806480u);
        hi = hsub2(__byte_perm(w, 0x64646464u, 0x4342), 0x64806480u);
    } else {
        lo = e4m3x2_f16x2((uint16_t)w);
        hi = e4m3x2_f16x2((uint16_t)(w >> 16));
    }
}

} // namespace b200
