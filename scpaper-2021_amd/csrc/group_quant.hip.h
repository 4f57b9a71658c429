// Quantising groups of binary16 values to 4 or 8 bits with a binary16 scale and lowest value: what the cache of keys and values
// (kv_cache.hip) and the 4-bit weights (w4.hip) share.
//
// A group [low, high] gets the smallest binary16 scale s with L * s >= high - low (L = 15 or 255), a value x the step nearest to
// (x - low) / s, ties to even.  Both are decided exactly: binary16 inputs lie on coarse grids, so quotients that fall on the border of two
// steps are common (5e-4 of the values of a normal distribution) and a rounded reciprocal would send them either way.
#pragma once
#include "common.hip.h"

namespace et {

__device__ __forceinline__ float f16_bits_value(unsigned bits) { return (float)__builtin_bit_cast(_Float16, (unsigned short)bits); }

// Bits of the smallest binary16 number s with levels * s >= high - low.  The difference of two binary16 numbers has up to 41 bits: it is
// held as r + e.  The quotient rounded to binary16 is next to the answer or is it; levels * s has at most 19 bits and, near r, its
// difference from r is exact.
template <int LEVELS> __device__ __forceinline__ unsigned group_scale_bits(float low, float high) {
    constexpr float levels = LEVELS;
    const float r = high - low;
    const float took = r - high, e = (high - (r - took)) + (-low - took);  // high - low = r + e, after Knuth's two-sum
    unsigned b = __builtin_bit_cast(unsigned short, (_Float16)(r * (1.0f / levels)));
    if (b > 0 && __builtin_fmaf(levels, f16_bits_value(b - 1), -r) >= e) b--;
    if (__builtin_fmaf(levels, f16_bits_value(b), -r) < e) b++;
    return b;
}

// The step nearest to (x - low) / s; inv = 1 / s to an ulp or two (0 where s is 0).  The quotient is corrected once, which rounds it as a division would, and then to a whole number, ties
// to even.  Where x - low is exact in binary32 that is the exact decision: with all values multiples of u and high - low <= 2^24 u, a quotient that is not on the border of
// two steps is at least u / s >= (L - 1) 2^-24 from it (or 2^-12, what s is a multiple of), more than half of its last place, 2^-21 below 16 and 2^-17 below 256.
__device__ __forceinline__ float nearest_step(float x, float low, float s, float inv) {
    const float d = x - low, q = d * inv;
    return __builtin_rintf(__builtin_fmaf(__builtin_fmaf(-q, s, d), inv, q));
}

// The same where x - low may be rounded: next to a border the remainder in binary64, which is exact, decides.
__device__ __forceinline__ float nearest_step_wide(float x, float low, float s, float inv) {
    const float t = (x - low) * inv;
    float c = __builtin_rintf(t);
    if (fabsf(t - c) >= 0.5f - 0x1p-12f) {
        const double rest = ((double)x - (double)low) - (double)c * (double)s, half = 0.5 * (double)s;
        const bool odd = ((int)c & 1) != 0;
        if (rest > half || (rest == half && odd)) c += 1.0f;
        else if (rest < -half || (rest == -half && odd)) c -= 1.0f;
    }
    return c;
}

// The smallest and the largest of eight values, as (smallest, -largest) in one word (so that a packed minimum folds both across lanes); NaN and infinities show in
// `magnitude`, the largest of their bits without the sign in either half.  tiny: the smallest of those bits less one (of no number but zero: 0xffff), in either half.
__device__ __forceinline__ h2 extremes(const h8 x, unsigned &magnitude, unsigned &tiny) {
    typedef unsigned short s2 __attribute__((ext_vector_type(2)));
    const h2 p[4] = {h2{x[0], x[1]}, h2{x[2], x[3]}, h2{x[4], x[5]}, h2{x[6], x[7]}};
    h2 lo = p[0], hi = p[0];
    s2 m = __builtin_bit_cast(s2, p[0]) & (unsigned short)0x7fff, t = m - (unsigned short)1;
#pragma unroll
    for (int i = 1; i < 4; i++) {
        lo = __builtin_elementwise_min(lo, p[i]);
        hi = __builtin_elementwise_max(hi, p[i]);
        const s2 bits = __builtin_bit_cast(s2, p[i]) & (unsigned short)0x7fff;
        m = __builtin_elementwise_max(m, bits);
        t = __builtin_elementwise_min(t, s2(bits - (unsigned short)1));
    }
    magnitude = __builtin_bit_cast(unsigned, m);
    tiny = __builtin_bit_cast(unsigned, t);
    return h2{lo[0] < lo[1] ? lo[0] : lo[1], -(hi[0] > hi[1] ? hi[0] : hi[1])};
}
__device__ __forceinline__ void extremes_of(h2 &e, unsigned &magnitude, h2 f, unsigned n) {
    typedef unsigned short s2 __attribute__((ext_vector_type(2)));
    e = __builtin_elementwise_min(e, f);
    magnitude = __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(s2, magnitude), __builtin_bit_cast(s2, n)));
}
__device__ __forceinline__ unsigned least_of(unsigned a, unsigned b) {
    typedef unsigned short s2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_elementwise_min(__builtin_bit_cast(s2, a), __builtin_bit_cast(s2, b)));
}
template <int CTRL> __device__ __forceinline__ void extremes_across(h2 &e, unsigned &magnitude) {
    const auto move = [](unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false); };
    extremes_of(e, magnitude, __builtin_bit_cast(h2, move(__builtin_bit_cast(unsigned, e))), move(magnitude));
}

// Codes of N eights of values of a group whose extremes are known, and the group's (scale, low).  tiny: as above, of these values.
template <int BITS, int N>
__device__ __forceinline__ void quantise(unsigned (&codes)[N * BITS / 4], unsigned &scale_low, const h8 (&x)[N], h2 extreme, unsigned magnitude, unsigned tiny) {
    const bool finite = (magnitude & 0xffffu) < 0x7C00u && magnitude >> 16 < 0x7C00u;
    const float lo = finite ? (float)extreme[0] : 0.0f, hi = finite ? -(float)extreme[1] : 0.0f;
    const unsigned sb = group_scale_bits<(1 << BITS) - 1>(lo, hi);
    const float s = f16_bits_value(sb), inv = s > 0.0f ? __builtin_amdgcn_rcpf(s) : 0.0f;
    // All are multiples of 2^(e - 25), e the exponent's bits of the smallest number other than zero among these values and the lowest: differences are exact up to 2^(e - 1).
    // Beyond, those of values within 2^-12 of the reach from zero may be rounded, and these lie within L 2^-12 steps of where zero does: of no concern unless zero itself is
    // next to a border, or the lowest value is that small.
    constexpr float kLevels = (1 << BITS) - 1;
    const float reach = hi - lo, zero_at = -lo * inv;
    const auto exact_to = [](unsigned bits) { return __builtin_ldexpf(1.0f, (int)max(bits >> 10, 1u) - 1); };
    const unsigned lo_bits = __builtin_bit_cast(unsigned short, (_Float16)lo) & 0x7fffu;
    const bool rounded = reach > exact_to(min(tiny & 0xffffu, tiny >> 16) + 1u) && fabsf(zero_at - __builtin_rintf(zero_at)) >= 0.5f - (kLevels + 1.0f) * 0x1p-12f;
    float c[8 * N];
    if (!(rounded || (lo_bits != 0 && reach > exact_to(lo_bits)))) {
#pragma unroll
        for (int i = 0; i < 8 * N; i++) c[i] = nearest_step((float)x[i / 8][i % 8], lo, s, inv);
    } else {
#pragma unroll
        for (int i = 0; i < 8 * N; i++) c[i] = nearest_step_wide((float)x[i / 8][i % 8], lo, s, inv);
    }
    // codes of 16 bits at a time are whole numbers of binary32
#pragma unroll
    for (int w = 0; w < N * BITS / 4; w++) {
        unsigned part[2];
#pragma unroll
        for (int p = 0; p < 2; p++) {
            constexpr int kPer = 16 / BITS;
            float sum = c[(2 * w + p) * kPer + kPer - 1];
#pragma unroll
            for (int i = kPer - 2; i >= 0; i--) sum = __builtin_fmaf(sum, (float)(1 << BITS), c[(2 * w + p) * kPer + i]);
            part[p] = (unsigned)sum;
        }
        codes[w] = finite ? part[0] | part[1] << 16 : 0;
    }
    scale_low = sb | (finite ? (unsigned)__builtin_bit_cast(unsigned short, (_Float16)lo) : 0x7E00u) << 16;
}

// What a code stands for, in binary16: rounding a group's scale up can carry its last steps beyond the largest number.
__device__ __forceinline__ _Float16 step_value(float c, float low, float s) {
    const float v = __builtin_fmaf(s, c, low);
    return (_Float16)(v > 65504.0f ? 65504.0f : v);  // (a NaN passes)
}

}  // namespace et
