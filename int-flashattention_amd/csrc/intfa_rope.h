// Rotary positions: the angle of a pair, and the rotation of the sixteen elements that one thread takes.
#pragma once
#include "intfa_device.h"

namespace intfa {

struct RopeArgs {
    const double* freqs;          // radians per position of each pair; nullptr: no rotation
    int32_t pairs, interleaved;
    float magnitude;
};

// magnitude * (cos, sin) of position * freq.  The angle is formed in turns and reduced in fp64: 2^31 positions at one radian each are
// 3.4e8 turns, of which two products and the constant's rounding lose up to 1.1e-7 of a turn (fp32 would have lost the turn itself at 1.7e7).  position: a
// whole number (rows count on from a first position of 32 bits, past those too).
__device__ __forceinline__ void rope_angle(double freq, double position, float magnitude, float& c, float& s) {
    double t = position * freq * 0.15915494309189533577;      // 1 / (2 pi)
    t -= __builtin_rint(t);
    sincospif(2.0f * (float)t, &s, &c);
    c *= magnitude;
    s *= magnitude;
}
// (a, b) turned (the compiler fuses one product of each sum into it: at most two roundings)
__device__ __forceinline__ void rope_turn(float& a, float& b, float c, float s) {
    const float x = a * c - b * s;
    b = b * c + a * s;
    a = x;
}

// A row of D elements in units of sixteen.  Rotated units hold eight pairs: elements 8 u .. and pairs + 8 u .. of the half layout, 16 u ..
// interleaved.  The elements behind the pairs are units of sixteen in order.  Returns the first elements of the unit's two groups of eight.
__device__ __forceinline__ void rope_unit(int u, int pairs, bool interleaved, int& first, int& second) {
    const bool half = 8 * u < pairs && !interleaved;
    first = half ? 8 * u : 16 * u;
    second = half ? pairs + 8 * u : 16 * u + 8;
}
// x: the two groups of eight of rotated unit u, c and s its eight angles.
__device__ __forceinline__ void rope_turn_unit(float (&x)[16], const float (&c)[8], const float (&s)[8], bool interleaved) {
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 8; ++i) rope_turn(x[2 * i], x[2 * i + 1], c[i], s[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) rope_turn(x[i], x[8 + i], c[i], s[i]);
    }
}

// ---- 16-bit groups of eight
template <int DT> __device__ __forceinline__ void unpack8(const v4i raw, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = (uint32_t)raw[i];
        if (DT == 0) {
            x[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w & 0xffffu));
            x[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
        } else {
            x[2 * i] = __builtin_bit_cast(float, w << 16);
            x[2 * i + 1] = __builtin_bit_cast(float, w & 0xffff0000u);
        }
    }
}
template <int DT> __device__ __forceinline__ v4i pack8(const float* x) {
    v4i r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint16_t lo, hi;
        if (DT == 0) {
            lo = __builtin_bit_cast(uint16_t, (_Float16)x[2 * i]);
            hi = __builtin_bit_cast(uint16_t, (_Float16)x[2 * i + 1]);
        } else {
            lo = (uint16_t)f32_to_bf16(x[2 * i]);
            hi = (uint16_t)f32_to_bf16(x[2 * i + 1]);
        }
        r[i] = (int)((uint32_t)hi << 16 | lo);
    }
    return r;
}

}  // namespace intfa
