// Eight neighbouring elements at a time: 16-bit tensors move 16 bytes per access, f32 tensors 32,
// 8-bit codes 8.  The element type is a run-time value; the switch is uniform over the grid and
// costs a few instructions per eight elements.
#pragma once

#include "common.cuh"

namespace b200 {

__device__ __forceinline__ float2 bf16x2_to_f32(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ float2 f16x2_to_f32(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }

// ptr: the first of the eight; aligned to their size together (16 bytes for 8 and 16-bit types too)
__device__ __forceinline__ void load8(int dt, const void *ptr, float (&v)[8]) {
    if (dt == B200_DT_F32) {
        const float4 a = ((const float4 *)ptr)[0], b = ((const float4 *)ptr)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        return;
    }
    const uint4 u = *(const uint4 *)ptr;
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if (dt == B200_DT_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = bf16x2_to_f32(w[i]);
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = f16x2_to_f32(w[i]);
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
    }
}

// plain roundings to nearest even (bf16 keeps denormals)
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void store8(int dt, void *ptr, const float (&v)[8]) {
    if (dt == B200_DT_F32) {
        ((float4 *)ptr)[0] = make_float4(v[0], v[1], v[2], v[3]);
        ((float4 *)ptr)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else if (dt == B200_DT_BF16) {
        *(uint4 *)ptr = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    } else {
        *(uint4 *)ptr = make_uint4(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]), pack_f16x2(v[4], v[5]), pack_f16x2(v[6], v[7]));
    }
}
__device__ __forceinline__ void store1(int dt, void *ptr, int64_t i, float v) {
    if (dt == B200_DT_F32) ((float *)ptr)[i] = v;
    else if (dt == B200_DT_BF16) ((uint16_t *)ptr)[i] = (uint16_t)pack_bf16x2(v, 0.f);
    else ((uint16_t *)ptr)[i] = (uint16_t)pack_f16x2(v, 0.f);
}

// ---- 8-bit codes of a value in units of its scale ------------------------------------------
// s8 is held to +-127, so that a code and its negative both exist; e4m3 to +-448.  The factor
// of the scale, 1 / 127 or 1 / 448 rounded to f32, multiplies the largest magnitude.
__device__ __forceinline__ float code_peak_factor(int dt) { return dt == B200_DT_S8 ? 1.f / 127.f : 1.f / 448.f; }
// the smallest scale: its reciprocal, 2^126, is still finite, so that rows of zeros (and of
// values next to them) need no special case
constexpr float CODE_SCALE_MIN = 1.17549435e-38f; // 2^-126

// The caller's values lie within the peak already, up to a rounding (a row or page times the reciprocal of its own
// scale; `held` below for the others).  s8: adding 1.5 * 2^23 rounds to the nearest integer, ties to even, and leaves it in the
// low byte -- on the ordinary f32 pipe, where a conversion instruction runs at an eighth of the rate.
__device__ __forceinline__ uint32_t round_s8(float v) { return __float_as_uint(__fadd_rn(v, 12582912.f)); }
__device__ __forceinline__ float held(int dt, float v) { // to the peak; NaN is not for here
    const float peak = dt == B200_DT_S8 ? 127.f : 448.f;
    return fminf(fmaxf(v, -peak), peak);
}
// two values, the first in the low byte; rounded once, held to +-448, NaN is 0x7f
__device__ __forceinline__ uint32_t code_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t codes4(int dt, float a, float b, float c, float d) {
    if (dt == B200_DT_S8)
        return __byte_perm(__byte_perm(round_s8(a), round_s8(b), 0x0040), __byte_perm(round_s8(c), round_s8(d), 0x0040), 0x5410);
    return code_e4m3x2(a, b) | code_e4m3x2(c, d) << 16;
}
__device__ __forceinline__ uint8_t code1(int dt, float v) {
    return dt == B200_DT_S8 ? (uint8_t)round_s8(v) : (uint8_t)code_e4m3x2(v, 0.f);
}
__device__ __forceinline__ float code_value(int dt, uint8_t c) { return dt == B200_DT_S8 ? (float)(int8_t)c : e4m3_to_f32(c); }
// the four codes of a word
__device__ __forceinline__ void code_values4(int dt, uint32_t w, float (&v)[4]) {
    if (dt == B200_DT_S8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) // code + 128 in the low byte of 2^23, minus 2^23 + 128: exact
            v[i] = __uint_as_float(__byte_perm(w ^ 0x80808080u, 0x4b000000u, 0x7540 + i)) - 8388736.f;
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * i)), __NV_E4M3);
            const float2 f = __half22float2(__half2(h));
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
    }
}

// maximum that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

} // namespace b200
