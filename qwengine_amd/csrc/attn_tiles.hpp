// MFMA helpers and the format of 16-bit partial states, which the prefill kernels and the batched decode have in common.
#pragma once

#include "kv_operands.hpp"
#include "pf_plan.hpp"

namespace qwa {

constexpr float PF_LOG2E = 1.4426950408889634f;

__device__ __forceinline__ h8 lds_h8(const _Float16* p) { return *reinterpret_cast<const h8*>(p); }

// max of three floats in one instruction (fmaxf would first canonicalize each MFMA result; scores are never sNaN)
__device__ __forceinline__ float max3f(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// max / sum over the four 16-lane rows of the wave (lanes l, l ^ 16, l ^ 32, l ^ 48) with the gfx950 lane swaps:
// permlane16_swap(x, x) leaves row pairs {r0, r0, r2, r2} / {r1, r1, r3, r3}, permlane32_swap {lo, lo} / {hi, hi}
__device__ __forceinline__ float rows_max(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    float y;
    asm("v_max_f32 %0, %1, %2" : "=v"(y) : "v"(__uint_as_float(a[0])), "v"(__uint_as_float(a[1])));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    asm("v_max_f32 %0, %1, %2" : "=v"(y) : "v"(__uint_as_float(b[0])), "v"(__uint_as_float(b[1])));
    return y;
}
__device__ __forceinline__ float rows_sum(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float y = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// 16-bit partials: O / l of a (split, row) as signed 16-bit fixed point against the row's largest |O / l| (the scale
// s = max / 32767 goes with (m, l)): absolute error <= s / 2 = max |O / l| * 2^-16 per value.
__device__ __forceinline__ int pf_q16(float v) { return (int)fminf(fmaxf(__builtin_rintf(v), -32767.0f), 32767.0f); }
__device__ __forceinline__ uint2 pack16x4(float a, float b, float c, float d) {
    return make_uint2(((uint32_t)pf_q16(a) & 0xFFFFu) | ((uint32_t)pf_q16(b) << 16),
                      ((uint32_t)pf_q16(c) & 0xFFFFu) | ((uint32_t)pf_q16(d) << 16));
}
__device__ __forceinline__ float4 unpack16x4(uint2 w) {
    return make_float4((float)(int16_t)(w.x & 0xFFFFu), (float)(int16_t)(w.x >> 16), (float)(int16_t)(w.y & 0xFFFFu),
                       (float)(int16_t)(w.y >> 16));
}
using PfPartO = uint2;    // four 16-bit values
using PfPartMl = float4;  // (m, l, scale, unused)

}  // namespace qwa
