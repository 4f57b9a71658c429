// Quantising groups of binary16 values to 4 or 8 bits with a binary16 scale and lowest value: what the cache of keys and values
// (kv_cache.hip) and the 4-bit weights (w4.hip) share.
//
// A group [low, high] gets the smallest binary16 scale s with L * s >= high - low (L = 15 or 255), a value x the step nearest to
// (x - low) / s, ties to even.  Both are decided exactly: binary16 inputs lie on coarse grids, so quotients that fall on the border of two
// steps are common (5e-4 of the values of a normal distribution) and a rounded reciprocal would send them either way.
#pragma once
#include "common.hip.h"

namespace et {

constexpr int kRowRor4 = 0x124, kRowRor8 = 0x128;

__device__ __forceinline__ float f16_bits_value(unsigned bits) { return (float)__builtin_bit_cast(_Float16, (unsigned short)bits); }

// Bits of the smallest binary16 number s with levels * s >= high - low.  The difference of two binary16 numbers has up to 41 bits: it is
// held as r + e.  The quotient rounded to binary16 is next to the answer or is it; levels * s has at most 19 bits and, near r, its
// difference from r is exact.
__device__ __forceinline__ unsigned group_scale_bits(float low, float high, float levels) {
    const float r = high - low;
    const float took = r - high, e = (high - (r - took)) + (-low - took);  // high - low = r + e, after Knuth's two-sum
    unsigned b = __builtin_bit_cast(unsigned short, (_Float16)(r / levels));
    if (b > 0 && levels * f16_bits_value(b - 1) - r >= e) b--;
    if (levels * f16_bits_value(b) - r < e) b++;
    return b;
}

// The step nearest to (x - low) / s; inv = 1 / s to an ulp or two (any finite number where s is 0).  The quotient in binary32 is off by less than 1e-4 steps,
// so it decides everywhere but next to a border, where the remainder in binary64, which is exact, does.
__device__ __forceinline__ float nearest_step(float x, float low, float s, float inv) {
    const float d = x - low;
    float c = __builtin_rintf(d * inv);
    const float r = __builtin_fmaf(-c, s, d);
    if (fabsf(2.0f * fabsf(r) - s) <= s * 0x1p-12f) {
        const double rest = ((double)x - (double)low) - (double)c * (double)s, half = 0.5 * (double)s;
        const bool odd = ((int)c & 1) != 0;
        if (rest > half || (rest == half && odd)) c += 1.0f;
        else if (rest < -half || (rest == -half && odd)) c -= 1.0f;
    }
    return c;
}

// What a code stands for, in binary16: rounding a group's scale up can carry its last steps beyond the largest number.
__device__ __forceinline__ _Float16 step_value(float c, float low, float s) {
    const float v = __builtin_fmaf(s, c, low);
    return (_Float16)(v > 65504.0f ? 65504.0f : v);  // (a NaN passes)
}

}  // namespace et
