// Rounding to int8 that the appends share.
#pragma once
#include "intfa_device.h"

namespace intfa {

constexpr float kLeastScale = 0x1p-100f;

__device__ __forceinline__ float finite_magnitude(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.f;      // (false for NaN too)
}
// rint(x / scale) within +-127, 0 for NaN, as a byte
__device__ __forceinline__ uint32_t quantise(float x, float scale) {
    const float q = rintf(x / scale);
    return (uint32_t)(q >= 127.f ? 127 : q <= -127.f ? -127 : q == q ? (int)q : 0) & 0xffu;
}
// Four of them for finite x with |x| <= 127 scale (to rounding).  The quotient is the correctly rounded one, by Markstein's correction of the product with
// the reciprocal (short of divisors whose significand is all ones, where it may be its neighbour); adding 1.5 * 2^23 rounds it to an integer
// in the low byte.  NaN gives 0: its low byte is.
__device__ __forceinline__ uint32_t quantise_low_byte(float x, float scale, float reciprocal) {
    const float q = x * reciprocal, e = __builtin_fmaf(-q, scale, x);
    return __builtin_bit_cast(uint32_t, __builtin_fmaf(e, reciprocal, q) + 12582912.0f);
}
__device__ __forceinline__ uint32_t quantise4(const float* x, float scale, float reciprocal) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = quantise_low_byte(x[i], scale, reciprocal);
    return __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u) | __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
}

}  // namespace intfa
