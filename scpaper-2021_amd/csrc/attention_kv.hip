// Attention over a cache of keys and values in 4 or 8 bits (layout: et_abi.h).
#include <math.h>

#include <algorithm>

#include "group_quant.hip.h"

namespace et {

int kv_check_cache(const char *fn, const et_kv_cache *c, const int32_t *table, int max_pages, int B, int n);

struct KvMhaArgs {
    const char *k_codes, *v_codes;
    const unsigned *k_scales, *v_scales;  // scale in the low half, low in the high one
    const int32_t *counts;
    const _Float16 *Q;
    _Float16 *Z;
    float *parts;         // of every (split, unit): stats [16][2], then values [rows of a block][hd]
    int ldq, ldz;
    int nkv, per, page, npages;
    int n, causal;
    int hd, cols, block_rows;  // columns of statistics a query row has, query rows of a workgroup
    int units, splits;    // (sequence, key/value head) pairs; workgroups that share the keys of one
    float scale_log2e;
};

// What the first requests need stands in front, in registers when a wave starts (14 words are):
//   splits   workgroups that share the keys of a (sequence, key/value head), units such pairs; per   query heads of one
//   magic, shift   pieces of 16 keys to pages: piece / (page / 16) = piece * magic >> shift
#define KV_LEADING const int32_t *table_at, const int32_t *starts_at, const int32_t *counts_at, int max_pages, int units, int splits, int per, unsigned magic, unsigned shift, \
                   int page_pieces, int n

typedef unsigned u2 __attribute__((ext_vector_type(2), aligned(4)));
typedef unsigned u3 __attribute__((ext_vector_type(3), aligned(4)));
typedef unsigned u4 __attribute__((ext_vector_type(4), aligned(4)));

// N consecutive words.
template <int N> __device__ __forceinline__ void load_words(unsigned (&to)[N], const char *from) {
    constexpr int kWhole = N / 4 * 4;
#pragma unroll
    for (int i = 0; i < kWhole; i += 4) {
        const u4 v = *reinterpret_cast<const u4 *>(from + i * 4);
        to[i] = v[0], to[i + 1] = v[1], to[i + 2] = v[2], to[i + 3] = v[3];
    }
    if constexpr (N % 4 == 3) {
        const u3 v = *reinterpret_cast<const u3 *>(from + kWhole * 4);
        to[kWhole] = v[0], to[kWhole + 1] = v[1], to[kWhole + 2] = v[2];
    } else if constexpr (N % 4 == 2) {
        const u2 v = *reinterpret_cast<const u2 *>(from + kWhole * 4);
        to[kWhole] = v[0], to[kWhole + 1] = v[1];
    } else if constexpr (N % 4 == 1) {
        to[kWhole] = *reinterpret_cast<const unsigned *>(from + kWhole * 4);
    }
}

template <int BITS, int HD> struct KvShape {
    static constexpr int kGroups = HD / 32;
    static constexpr int kCols = kGroups == 1 ? 1 : kGroups == 2 ? 2 : kGroups <= 4 ? 4 : 8;  // columns of a query row
    static constexpr int kRows = 16 / kCols;                                                   // query rows of a block
    static constexpr int kTokenBytes = HD * BITS / 8;
    static constexpr int kKeyWords = kTokenBytes / 16;  // of a lane: a quarter of a key
    static constexpr int kPieces = HD / 32;             // of eight channels in that quarter
    static constexpr int kUnits = HD * BITS / 16 / 16;  // whole units of 16 bits of a value that a lane has
    static constexpr bool kHalfUnit = HD * BITS / 16 % 16 != 0;  // and two channels of one that two lanes share
    static constexpr int kValueWords = 2 * kUnits + 2 * kHalfUnit;
    static constexpr int kUnitChannels = 16 / BITS;
    static constexpr int kAcc = HD / 16;
    static constexpr int kPart = 32 + kRows * HD;  // floats that a workgroup leaves
};

constexpr float kNothing = -1e30f;

// Weights of channel groups that share a reference: a group whose scales are far smaller than another's would have its weights among the subnormal binary16
// numbers, where the second number of a weight holds nothing (300 keys, scales 2^20 apart: 3.5e-4 of the group's 2-norm instead of 2.1e-4, 2^22: 9e-4).  Where scales are more than 2^kLeastLift
// apart, a group's weights, and with them its products, are times 2^lift: 15 is enough, since scales reach from 2^-24 to 2^13 and weights keep their bits 2^16 below the largest.
constexpr float kMostLift = 15.0f, kLeastLift = 8.0f;

// The lift of a group, at most 15, whose largest p * scale is below 2^reach: to 2^11 where lifts are chosen, else no more than keeps it at 2^15.
__device__ __forceinline__ float next_lift(float lift, float reach, float most, bool choose) {
    return fmaxf(fminf(choose ? floorf(11.0f - reach) : fminf(lift, floorf(15.0f - reach)), most), 0.0f);
}

#define ET_KV_CONST(T, p) ((const __attribute__((address_space(4))) T *)(p))

__device__ __forceinline__ h8 as_h8(unsigned a, unsigned b, unsigned c, unsigned d) {
    typedef unsigned w4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(h8, w4{a, b, c, d});
}
__device__ __forceinline__ float low_half(unsigned w) { return (float)__builtin_bit_cast(h2, w)[0]; }
__device__ __forceinline__ float high_half(unsigned w) { return (float)__builtin_bit_cast(h2, w)[1]; }

// Codes of a value's unit, taken from both halves of a word, as subnormal binary16 numbers.  The products lose what lies some 2^-24 under the largest's place, and a code in the
// lowest bits of a half, where it stands 2^10 under that place, cost results 3e-4 of themselves where the values' sum nearly cancels (131071 keys): the codes
// are moved up.  4 bits: bits 3 to 6 (codes 0 and 1, code * 2^-21) and 7 to 10 (2 and 3, * 2^-17; bit 10 is the lowest of the exponent, where the numbers still are as far
// apart), three shifts and four masks a word; 8 bits: bits 2 to 9 (* 2^-22).
template <int BITS> constexpr float code_unit(int k) { return BITS == 8 ? 0x1p22f : k < 2 ? 0x1p21f : 0x1p17f; }
template <int BITS> __device__ __forceinline__ unsigned raised(unsigned w, int k) {
    if constexpr (BITS == 8) return (k == 0 ? w << 2 : w >> 6) & 0x03fc03fcu;
    return k == 0 ? (w << 3) & 0x00780078u : k == 1 ? (w >> 1) & 0x00780078u : k == 2 ? (w >> 1) & 0x07800780u : (w >> 5) & 0x07800780u;
}

// A row's result: zero where it sees nothing; at most binary16's largest number, since it is the rounding up of a group's scale alone that can carry it beyond (as in step_value).
__device__ __forceinline__ _Float16 result_value(float sum, float l) {
    const float v = l == 0.0f ? 0.0f : sum / l;
    return (_Float16)(v > 65504.0f ? 65504.0f : v);  // (a NaN passes)
}

// Sum over the kCols neighbouring lanes of a query row.
template <int COLS> __device__ __forceinline__ float cols_sum(float v) {
    if constexpr (COLS >= 2) v += dpp_move<kDppQuadXor1>(v);
    if constexpr (COLS >= 4) v += dpp_move<kDppQuadXor2>(v);
    if constexpr (COLS >= 8) v += dpp_move<0x141>(v);  // row_half_mirror
    return v;
}

// Eight channels of a key as subnormal numbers, code * 2^-key_unit_log2, every other one * 16 for 4 bits: channels 0 4 1 5 2 6 3 7, or 0 2 1 3 4 6 5 7.  As in values, codes in the lowest bits
// would cost the smaller terms of a score theirs: 4-bit codes are in bits 3 to 6 and 7 to 10 (at 0 to 3 and 4 to 7, one instruction less in six, a query's channel 100 times the others, and small in the
// keys, made 2.1e-4 of the result's 2-norm 2.6e-4 to 3.7e-4).
template <int BITS> constexpr int key_unit_log2() { return BITS == 4 ? 21 : 24; }
template <int BITS> __device__ __forceinline__ h8 key_codes(const unsigned *w) {
    if constexpr (BITS == 4) {
        const unsigned x = w[0] << 3, y = w[0] >> 5;
        return as_h8(x & 0x00780078u, x & 0x07800780u, y & 0x00780078u, y & 0x07800780u);
    } else {
        return as_h8(w[0] & 0x00ff00ffu, (w[0] >> 8) & 0x00ff00ffu, w[1] & 0x00ff00ffu, (w[1] >> 8) & 0x00ff00ffu);
    }
}

// The same eight channels of a query times `grow`, 1 / 16 of that where the code comes out 16-fold; their sum goes to `sum`.
template <int BITS> __device__ __forceinline__ h8 query_order(h8 x, float grow, float &sum) {
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
        f[k] = grow != 0.0f ? (float)x[k] * grow : 0.0f;
        sum += f[k];
    }
    if constexpr (BITS == 4)
        return h8{(_Float16)f[0], (_Float16)f[4], (_Float16)(f[1] / 16), (_Float16)(f[5] / 16), (_Float16)f[2], (_Float16)f[6], (_Float16)(f[3] / 16), (_Float16)(f[7] / 16)};
    else
        return h8{(_Float16)f[0], (_Float16)f[2], (_Float16)f[1], (_Float16)f[3], (_Float16)f[4], (_Float16)f[6], (_Float16)f[5], (_Float16)f[7]};
}

// What a row of Q is multiplied by.  Scores of a row with an infinity are infinite of either sign or NaN, and have no softmax: it becomes NaN here, or the weights of
// scores that are all minus infinity would add up to nothing, as where a row sees no key.
__device__ __forceinline__ float query_growth(float top, int up, float scale) {
    return top <= 65504.0f ? __builtin_ldexpf(scale < 0.0f ? -1.0f : 1.0f, up) : __builtin_nanf("");
}

// p * scale as two binary16 numbers: rounded to one, whose error is relative to a value's height above the group's lowest, results were 2 to 3 times as far off as their own
// rounding (5.9e-4 against 2.1e-4, 2-norm, 131071 keys of random values).  With a zero that the compiler does not know each is one instruction, which widens, multiplies,
// adds and rounds.
__device__ __forceinline__ float hidden_zero() {
    float zero = 0.0f;
    asm("" : "+v"(zero));
    return zero;
}
// PAIRS: two weights are rounded in one instruction, from binary32, instead of each with its product (16 rows of heads of 128: 59.8 us instead of 60.7; four rows of
// 131071 keys the other way, 37.0 and 36.1).
template <bool PAIRS = false> __device__ __forceinline__ void weight_of(_Float16 &w, _Float16 &rest, float p, unsigned scale_low, float zero) {
    float whole = __builtin_fmaf(p, low_half(scale_low), zero);
    if constexpr (PAIRS) asm("" : "+v"(whole));
    w = (_Float16)whole;
    float part = __builtin_fmaf(p, low_half(scale_low), -(float)w);
    if constexpr (PAIRS) asm("" : "+v"(part));
    rest = (_Float16)part;
}

// acc += (w + rest) * codes over 32 keys, 4 j .. 4 j + 3 of two pieces.
template <int BITS, int HD> __device__ __forceinline__ void weigh_values(f4 *acc, h8 w, h8 rest, const unsigned *first, const unsigned *second, int c) {
    using S = KvShape<BITS, HD>;
    auto weigh = [&](int i, h8 codes) {
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, codes, acc[i], 0, 0, 0);
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(rest, codes, acc[i], 0, 0, 0);
    };
#pragma unroll
    for (int u = 0; u < S::kUnits; u++)
#pragma unroll
        for (int k = 0; k < S::kUnitChannels; k++)
            weigh(S::kUnitChannels * u + k, as_h8(raised<BITS>(first[2 * u], k), raised<BITS>(first[2 * u + 1], k), raised<BITS>(second[2 * u], k), raised<BITS>(second[2 * u + 1], k)));
    if constexpr (S::kHalfUnit) {
        // codes 2 (c % 2) and the next, moved to the places of codes 0 and 1
        const int shift = (c & 1) * 8;
        const unsigned a0 = first[2 * S::kUnits] >> shift, a1 = first[2 * S::kUnits + 1] >> shift;
        const unsigned b0 = second[2 * S::kUnits] >> shift, b1 = second[2 * S::kUnits + 1] >> shift;
#pragma unroll
        for (int k = 0; k < 2; k++) weigh(4 * S::kUnits + k, as_h8(raised<4>(a0, k), raised<4>(a1, k), raised<4>(b0, k), raised<4>(b1, k)));
    }
}

// The channel that column c of product i stands for.
template <int BITS, int HD> __device__ __forceinline__ int value_channel(int i, int c) {
    using S = KvShape<BITS, HD>;
    if (S::kHalfUnit && i >= S::kUnits * S::kUnitChannels) return 64 * S::kUnits + (c >> 1) * 4 + (c & 1) * 2 + i - S::kUnits * S::kUnitChannels;
    return (c * S::kUnits + i / S::kUnitChannels) * S::kUnitChannels + i % S::kUnitChannels;
}

// What its products are to be multiplied with.
template <int BITS, int HD> constexpr float value_unit(int i) {
    using S = KvShape<BITS, HD>;
    return code_unit<BITS>(i < S::kUnits * S::kUnitChannels ? i % S::kUnitChannels : 0);
}

// A lane's words of the values of 16 keys.
template <int BITS, int HD> __device__ __forceinline__ void load_value(unsigned *to, const char *units, const char *half_units) {
    using S = KvShape<BITS, HD>;
    unsigned whole[S::kUnits > 0 ? 2 * S::kUnits : 1], half[2];
    if constexpr (S::kUnits > 0) load_words<2 * S::kUnits>(whole, units);
    if constexpr (S::kHalfUnit) load_words<2>(half, half_units);
#pragma unroll
    for (int i = 0; i < 2 * S::kUnits; i++) to[i] = whole[i];
    if constexpr (S::kHalfUnit) to[2 * S::kUnits] = half[0], to[2 * S::kUnits + 1] = half[1];
}

// Several rows a key/value head: blocks of 16 / kCols query rows, whose (row, group) pairs fill the 16 columns of the products of a tile of 32 keys.
//
// Scores: keys are the rows of the products, so a lane ends with keys 4 j .. 4 j + 3 of both pieces for its column, and these are the very keys that it weighs as a row of the
// products with the values: nothing moves between lanes but the sum of a row's groups, and a maximum when the reference moves.
//
// One sequence of 131071 tokens, 32 heads over 8 of 128: 36.4 us, 4.6 TB/s, and 5 us to join 64 parts.  16 sequences of 1500, 8 heads of 96, 7 rows, 8 bits: 15 us, bound by 236
// vector instructions a tile on two waves a SIMD (a tile ahead in registers: 16.3, and 43 us in the first).
template <int BITS, int HD> constexpr int kv_rows_waves() { return HD == 32 ? 6 : HD == 64 ? (BITS == 4 ? 6 : 5) : HD <= 128 ? 4 : 2; }

template <int BITS, int HD, int NW> __global__ __launch_bounds__(NW * 64, (kv_rows_waves<BITS, HD>())) void mha_kv_kernel(KV_LEADING, const KvMhaArgs a) {
    using S = KvShape<BITS, HD>;
    constexpr int COLS = S::kCols, ROWS = S::kRows, G = S::kGroups, TB = S::kTokenBytes;
    __shared__ float lds_vals[NW][ROWS * HD];
    __shared__ float lds_stats[NW][3][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, j = lane >> 4;
    const int qh = c / COLS, gg = c % COLS;
    const int kv = blockIdx.x, b = blockIdx.y, nkv = gridDim.x;
    const int block = splits == 1 ? blockIdx.z : blockIdx.z / splits, split = blockIdx.z - block * splits;

    // as in mha_kv_few_kernel
    const auto *table = ET_KV_CONST(int32_t, table_at) + (size_t)b * max_pages;
    const int t_step = splits * NW;
    int t = split * NW + wave;
    const bool wide = (page_pieces & 1) == 0;
    int page[2], off[2];
    auto ask = [&](int tile) {
        const int piece = 2 * tile;
        int pidx = (int)(((unsigned long long)(unsigned)piece * magic) >> shift), at = piece - pidx * page_pieces;
        off[0] = at << 4;
        page[0] = pidx < max_pages ? table[pidx] : -1;
        if (wide) return;
        const bool on = ++at == page_pieces;
        off[1] = (on ? 0 : at) << 4;
        pidx += on;
        page[1] = pidx < max_pages ? table[pidx] : -1;
    };
    ask(t);

    // the rows of this block, and what they see
    const int start = starts_at ? ET_KV_CONST(int32_t, starts_at)[b] : 0;
    const int count = counts_at ? min(max(ET_KV_CONST(int32_t, counts_at)[b], 0), n) : n;
    const int row0 = block * ROWS, rows = min(ROWS, count * per - row0);
    if (rows <= 0) return;
    const long long most = (long long)max_pages * a.page;
    const int end = (int)min(max((long long)start + count, 0LL), most);
    auto row_of = [&](int row) { return n == 1 ? 0 : row / per; };  // of the call's rows
    auto limit = [&](int i) { return a.causal ? (int)min((long long)end, max((long long)start + i + 1, 0LL)) : end; };
    const int lim_least = limit(row_of(row0)), lim_most = limit(row_of(row0 + rows - 1));
    const int t_end = (lim_most + 31) >> 5;

    // Q in the order that the keys' codes come out of their words: 0 4 1 5 2 6 3 7 (4 bits, where 1 5 3 7 come out 16-fold) or 0 2 1 3 4 6 5 7; times a power of two
    // that brings a row's largest to 2^14 .. 2^15, so that the smaller ones keep their bits below 1 / 16; zero in the columns of the other groups
    h8 q[S::kPieces];
    const int row = row0 + min(qh, rows - 1), i_row = row_of(row), r_row = row - i_row * per;
    const int lim = limit(i_row);
    const _Float16 *qrow = a.Q + ((size_t)b * n + i_row) * a.ldq + (size_t)(kv * per + r_row) * HD + j * (HD / 4);
    float top = 0.0f, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < S::kPieces; i++) {
        q[i] = *reinterpret_cast<const h8 *>(qrow + 8 * i);
#pragma unroll
        for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf((float)q[i][e]));
    }
    top = rows_max(top);
    const int up = top > 0.0f ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
    const float grow = query_growth(top, up, a.scale_log2e);
    const float key_scale = __builtin_ldexpf(fabsf(a.scale_log2e), key_unit_log2<BITS>() - up);
#pragma unroll
    for (int i = 0; i < S::kPieces; i++) q[i] = query_order<BITS>(q[i], (j * (HD / 4) + 8 * i) / 32 == gg ? grow : 0.0f, sum);
    const float qsum = __builtin_ldexpf(rows_sum(sum), -key_unit_log2<BITS>());

    float ref = kNothing, l = 0.0f, z = 0.0f;
    f4 acc[S::kAcc];
#pragma unroll
    for (int i = 0; i < S::kAcc; i++) acc[i] = f4{0.f, 0.f, 0.f, 0.f};

    const unsigned key_at = c * TB + j * (TB / 4), value_at = j * (4 * TB) + c * (8 * S::kUnits), half_at = j * (4 * TB) + 128 * S::kUnits + (c >> 1) * 8;
    const char *k_codes = a.k_codes + (size_t)kv * a.page * TB, *v_codes = a.v_codes + (size_t)kv * a.page * TB;
    const unsigned *k_scales = a.k_scales + (size_t)kv * (G * a.page), *v_scales = a.v_scales + (size_t)kv * (G * a.page);
    const unsigned page_bytes = (unsigned)nkv * a.page * TB, page_scales = (unsigned)nkv * G * a.page, scales_at = (unsigned)(min(gg, G - 1) * a.page + 4 * j);

    const float zero = hidden_zero();
    for (; t < t_end; t += t_step) {
        // where the pieces lie; one that nobody sees, or without a page, is read from the place of the one before it
        size_t at[2], scale_at[2];
        bool ok[2];
        ok[0] = page[0] >= 0 && page[0] < a.npages;
        const unsigned from = ok[0] ? page[0] : 0, from_off = ok[0] ? off[0] : 0;
        at[0] = (size_t)from * page_bytes + from_off * TB;
        scale_at[0] = (size_t)from * page_scales + from_off + scales_at;
        if (wide) {
            ok[1] = ok[0];
            const bool second = t * 32 + 16 < lim_most;
            at[1] = at[0] + (second ? 16 * TB : 0);
            scale_at[1] = scale_at[0] + (second ? 16 : 0);
        } else {
            ok[1] = t * 32 + 16 < lim_most && page[1] >= 0 && page[1] < a.npages;
            const unsigned from1 = ok[1] ? page[1] : from, off1 = ok[1] ? off[1] : from_off;
            at[1] = (size_t)from1 * page_bytes + off1 * TB;
            scale_at[1] = (size_t)from1 * page_scales + off1 + scales_at;
        }
        unsigned kw[2][S::kKeyWords], vw[2][S::kValueWords];
        u4 ks[2], vs[2];
#pragma unroll
        for (int s = 0; s < 2; s++) {
            load_words<S::kKeyWords>(kw[s], k_codes + at[s] + key_at);
            ks[s] = *reinterpret_cast<const u4 *>(k_scales + scale_at[s]);
        }
#pragma unroll
        for (int s = 0; s < 2; s++) {
            vs[s] = *reinterpret_cast<const u4 *>(v_scales + scale_at[s]);
            load_value<BITS, HD>(vw[s], v_codes + at[s] + value_at, v_codes + at[s] + half_at);
        }
        const int tile = t * 32;
        const bool whole = tile + 32 <= lim_least && ok[0] && ok[1];
        const bool ok0 = ok[0], ok1 = ok[1];
        ask(t + t_step);

        float y[8];
#pragma unroll
        for (int s = 0; s < 2; s++) {
            f4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < S::kPieces; i++) {
                const h8 codes = key_codes<BITS>(&kw[s][i * BITS / 4]);
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, q[i], d, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; r++)
                y[4 * s + r] = cols_sum<COLS>(__builtin_fmaf(low_half(ks[s][r]), d[r], high_half(ks[s][r]) * qsum)) * key_scale;
        }
        if (!whole) {
            // (what a row does not see must not come into its sums, whatever it is: the lowest value of another row's key may be NaN, and 0 * NaN is)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int s = e >> 2, pos = tile + 16 * s + 4 * j + (e & 3);
                const bool there = s == 0 ? ok0 : ok1;
                vs[s][e & 3] = there && pos < lim ? vs[s][e & 3] : 0u;
                y[e] = there && pos < lim ? y[e] : kNothing;
            }
        }
        float most_s = low_half(vs[0][0]);
#pragma unroll
        for (int e = 1; e < 8; e++) most_s = fmaxf(most_s, low_half(vs[e >> 2][e & 3]));
        const float most_e = (float)__builtin_amdgcn_frexp_expf(most_s);
        h8 w, rest;
        float most_y = y[0];
#pragma unroll
        for (int e = 1; e < 8; e++) most_y = fmaxf(most_y, y[e]);
        // a weight is at most 2^15: p * scale < 2^(y - ref + exponent of the scale)
        const float reach = most_y + most_e;
        if (__any(reach > ref + 15.0f)) {
            const float next = fmaxf(ref, rows_max(reach) - 11.0f);
            const float f = __builtin_amdgcn_exp2f(ref - next);
            ref = next;
            l *= f;
            z *= f;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float fr = __shfl(f, 4 * j + r);
#pragma unroll
                for (int i = 0; i < S::kAcc; i++) acc[i][r] *= fr;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float p = y[e] == kNothing ? 0.0f : __builtin_amdgcn_exp2f(y[e] - ref);
            l += p;
            z = __builtin_fmaf(p, high_half(vs[e >> 2][e & 3]), z);
            _Float16 we, re;
            weight_of(we, re, p, vs[e >> 2][e & 3], zero);
            w[e] = we, rest[e] = re;
        }
        weigh_values<BITS, HD>(acc, w, rest, vw[0], vw[1], c);
    }

    // what the waves have, side by side
    const float ls = rows_sum(l), zs = rows_sum(z);
    if (j == 0) {
        lds_stats[wave][0][c] = ref;
        lds_stats[wave][1][c] = ls;
        lds_stats[wave][2][c] = zs;
    }
#pragma unroll
    for (int i = 0; i < S::kAcc; i++) {
        const int ch = value_channel<BITS, HD>(i, c);
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int row = 4 * j + r;
            if (row % COLS == ch >> 5) lds_vals[wave][row / COLS * HD + ch] = acc[i][r] * value_unit<BITS, HD>(i);
        }
    }
    __syncthreads();
    float *part = splits > 1 ? a.parts + ((size_t)blockIdx.z * units + (unsigned)(b * nkv + kv)) * S::kPart : nullptr;
    for (int e = threadIdx.x; e < rows * HD; e += NW * 64) {
        const int h = e / HD, ch = e - h * HD, col = h * COLS + (ch >> 5);
        float m = lds_stats[0][0][col];
#pragma unroll
        for (int w = 1; w < NW; w++) m = fmaxf(m, lds_stats[w][0][col]);
        float sum = 0.0f, ls = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = __builtin_amdgcn_exp2f(lds_stats[w][0][col] - m);
            sum = __builtin_fmaf(f, lds_vals[w][e] + lds_stats[w][2][col], sum);
            ls = __builtin_fmaf(f, lds_stats[w][1][col], ls);
        }
        if (part) {
            part[32 + e] = sum;
            if ((ch & 31) == 0) part[2 * col] = m, part[2 * col + 1] = ls;
        } else {
            const int row = row0 + h, i = row_of(row), r = row - i * per;
            a.Z[((size_t)b * n + i) * a.ldz + (size_t)(kv * per + r) * HD + ch] = result_value(sum, ls);
        }
    }
}

// Many rows: 16 query rows are the columns of the products, and the contraction is over one group at a time (P = 1).  P = 2: 8 rows, each in two columns, one for either of a
// pair of groups, half of each contraction's lanes with either; a row's weights are computed twice instead of, in mha_kv_kernel, four times.
//
// Scores: lane (c, j) needs eight channels of every group of key c, so the words of a key, loaded 16 bytes a lane, change places between the four rows of lanes (KvWords).
// Values: the 16 columns of a product are channels of one group, whose scale is in the rows' weights.
//
// Bound by its vector instructions, some 500 a tile of 16 rows and 32 keys of 128 channels (five a score and group, the rest the codes), next to 24 products: 64 sequences of
// 1000 tokens, 16 heads of 128, 16 rows 59 us (128 in blocks of 4), 8 of 4000, 4 heads, 256 rows 106 (195).  A spilled register a lane costs more than a wave a SIMD: at three
// of those, with spills, twice the time.
template <int BITS> struct KvWords {
    // Groups in fours, a two and a one: lane j loads what lies at j of a four's (two's, one's) bytes, group j of the four.
    static constexpr int W = BITS / 4;  // words of eight channels
    template <int G> static __device__ __forceinline__ void load(unsigned (&to)[G * W], const char *key, int j) {
        each<G>([&](auto n, int g) {
            constexpr int N = decltype(n)::value;
            unsigned v[N * W];
            load_words<N * W>(v, key + (g * 4 + j * N) * W * 4);
#pragma unroll
            for (int i = 0; i < N * W; i++) to[g * W + i] = v[i];
        });
    }
    // -> word w of group g at g * W + w, of the group's eights that of(G, g, j) names
    template <int G> static __device__ __forceinline__ void part(unsigned (&v)[G * W]) {
        auto swap32 = [](unsigned &p, unsigned &q) {
            auto r = __builtin_amdgcn_permlane32_swap(p, q, false, false);
            p = r[0], q = r[1];
        };
        auto swap16 = [](unsigned &p, unsigned &q) {
            auto r = __builtin_amdgcn_permlane16_swap(p, q, false, false);
            p = r[0], q = r[1];
        };
        each<G>([&](auto n, int g) {
#pragma unroll
            for (int w = 0; w < W; w++) {
                unsigned *x = v + g * W + w;
                if constexpr (decltype(n)::value == 4) {
                    swap32(x[0], x[2 * W]);
                    swap32(x[W], x[3 * W]);
                    swap16(x[0], x[W]);
                    swap16(x[2 * W], x[3 * W]);
                } else if constexpr (decltype(n)::value == 2) {
                    swap32(x[0], x[W]);
                }
            }
        });
    }
    // The eight channels (of four in a group) that lane j has of group g.
    static constexpr __device__ __forceinline__ int of(int G, int g, int j) { return g < G / 4 * 4 || G % 2 == 1 && g == G - 1 ? j : (j & 1) * 2 + (j >> 1); }

  private:
    template <int N> struct Number { static constexpr int value = N; };
    template <int G, typename F> static __device__ __forceinline__ void each(F f) {
#pragma unroll
        for (int g = 0; g + 4 <= G; g += 4) f(Number<4>(), g);
        if constexpr (G % 4 >= 2) f(Number<2>(), G / 4 * 4);
        if constexpr (G % 2 == 1) f(Number<1>(), G - 1);
    }
};

template <int BITS, int HD, int NW, int P> __global__ __launch_bounds__(NW * 64, (HD <= 64 ? 4 : 2)) void mha_kv_rows_kernel(KV_LEADING, const KvMhaArgs a) {
    constexpr int ROWS = 16 / P, G = HD / 32, SETS = G / P, PRODUCTS = 2 * P, VW = BITS == 8 ? 2 * P : 2, TB = HD * BITS / 8, W = BITS / 4;
    __shared__ float lds_vals[NW][ROWS * HD];
    __shared__ float lds_stats[NW][2 + SETS][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, j = lane >> 4;
    const int side = P == 2 ? c & 1 : 0;  // of a pair of groups
    const int kv = blockIdx.x, b = blockIdx.y, nkv = gridDim.x;
    const int block = splits == 1 ? blockIdx.z : blockIdx.z / splits, split = blockIdx.z - block * splits;

    // as in mha_kv_kernel
    const auto *table = ET_KV_CONST(int32_t, table_at) + (size_t)b * max_pages;
    const int t_step = splits * NW;
    int t = split * NW + wave;
    int page[2], off[2];
    auto ask = [&](int tile) {
        const int piece = 2 * tile;
        int pidx = (int)(((unsigned long long)(unsigned)piece * magic) >> shift), at = piece - pidx * page_pieces;
        off[0] = at << 4;
        page[0] = pidx < max_pages ? table[pidx] : -1;
        const bool on = ++at == page_pieces;
        off[1] = (on ? 0 : at) << 4;
        pidx += on;
        page[1] = pidx < max_pages ? table[pidx] : -1;
    };
    ask(t);

    const int start = starts_at ? ET_KV_CONST(int32_t, starts_at)[b] : 0;
    const int count = counts_at ? min(max(ET_KV_CONST(int32_t, counts_at)[b], 0), n) : n;
    const int row0 = block * ROWS, rows = min(ROWS, count * per - row0);
    if (rows <= 0) return;
    const long long most = (long long)max_pages * a.page;
    const int end = (int)min(max((long long)start + count, 0LL), most);
    auto row_of = [&](int row) { return n == 1 ? 0 : row / per; };  // of the call's rows
    auto limit = [&](int i) { return a.causal ? (int)min((long long)end, max((long long)start + i + 1, 0LL)) : end; };
    const int lim_least = limit(row_of(row0)), lim_most = limit(row_of(row0 + rows - 1));
    const int t_end = (lim_most + 31) >> 5;

    h8 q[G];
    float qsum[SETS];
    const int row = row0 + min(c / P, rows - 1), i_row = row_of(row), r_row = row - i_row * per;
    const int lim = limit(i_row);
    const _Float16 *qrow = a.Q + ((size_t)b * n + i_row) * a.ldq + (size_t)(kv * per + r_row) * HD;
    float top = 0.0f;
#pragma unroll
    for (int g = 0; g < G; g++) {
        q[g] = *reinterpret_cast<const h8 *>(qrow + (P == 2 ? ((g & ~1) + (j & 1)) * 32 + ((j >> 1) * 2 + (g & 1)) * 8 : g * 32 + KvWords<BITS>::of(G, g, j) * 8));
#pragma unroll
        for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf((float)q[g][e]));
    }
    top = rows_max(top);
    const int up = top > 0.0f ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
    const float grow = query_growth(top, up, a.scale_log2e);
    const float key_scale = __builtin_ldexpf(fabsf(a.scale_log2e), key_unit_log2<BITS>() - up);
#pragma unroll
    for (int g = 0; g < SETS; g++) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < P; i++) q[P * g + i] = query_order<BITS>(q[P * g + i], P == 1 || (j & 1) == side ? grow : 0.0f, sum);
        qsum[g] = __builtin_ldexpf(rows_sum(sum), -key_unit_log2<BITS>());
    }

    float ref = kNothing, l = 0.0f, z[SETS];
    f4 acc[SETS][PRODUCTS];
    unsigned lift = 0;    // of the sets, four bits each: what acc is times 2^ of
    bool lifted = false;  // any of any row
    auto lift_of = [](unsigned lifts, int g) { return (int)(lifts >> (4 * g) & 15u); };
#pragma unroll
    for (int g = 0; g < SETS; g++) {
        z[g] = 0.0f;
#pragma unroll
        for (int k = 0; k < PRODUCTS; k++) acc[g][k] = f4{0.f, 0.f, 0.f, 0.f};
    }

    // units of 16 bits of a value: 8 a group with 4 bits, of which two lanes take one, codes 0 and 1 or 2 and 3; 16 with 8 bits; of a pair of groups one or two a lane
    const unsigned key_at = c * TB + (P == 2 ? ((j & 1) * 4 + (j >> 1) * 2) * W * 4 : 0), value_at = j * (4 * TB) + (P == 2 ? c * (4 * VW) : (BITS == 4 ? c & 7 : c) * 8);
    const int code_at = P == 1 && BITS == 4 ? c & 8 : 0;
    const char *k_codes = a.k_codes + (size_t)kv * a.page * TB, *v_codes = a.v_codes + (size_t)kv * a.page * TB;
    const unsigned *k_scales = a.k_scales + (size_t)kv * (G * a.page), *v_scales = a.v_scales + (size_t)kv * (G * a.page);
    const unsigned page_bytes = (unsigned)nkv * a.page * TB, page_scales = (unsigned)nkv * G * a.page, scales_at = (unsigned)(side * a.page + 4 * j);

    constexpr bool kAtOnce = HD <= 128, kKeysAtOnce = HD <= 192;  // (the registers do not hold keys and values, or all keys, of wider heads)
    constexpr int kFirst = kKeysAtOnce ? SETS : 3;  // groups of the values that are asked for at once
    const float zero = hidden_zero();
    for (; t < t_end; t += t_step) {
        // where the pieces lie; one that nobody sees, or without a page, is read from the place of the one before it
        size_t at[2], scale_at[2];
        const bool ok0 = page[0] >= 0 && page[0] < a.npages, ok1 = t * 32 + 16 < lim_most && page[1] >= 0 && page[1] < a.npages;
        const unsigned from = ok0 ? page[0] : 0, from_off = ok0 ? off[0] : 0, from1 = ok1 ? page[1] : from, off1 = ok1 ? off[1] : from_off;
        at[0] = (size_t)from * page_bytes + from_off * TB;
        at[1] = (size_t)from1 * page_bytes + off1 * TB;
        scale_at[0] = (size_t)from * page_scales + from_off + scales_at;
        scale_at[1] = (size_t)from1 * page_scales + off1 + scales_at;
        unsigned kw[2][G * W], vw[2][SETS][VW];
        u4 ks[2][SETS], vs[2][SETS];
        auto load_keys = [&](int s) {
            if constexpr (P == 1) {
                KvWords<BITS>::template load<G>(kw[s], k_codes + at[s] + key_at, j);
            } else {
#pragma unroll
                for (int g = 0; g < SETS; g++) {
                    unsigned v[2 * W];
                    load_words<2 * W>(v, k_codes + at[s] + key_at + g * (8 * W * 4));
#pragma unroll
                    for (int i = 0; i < 2 * W; i++) kw[s][2 * W * g + i] = v[i];
                }
            }
#pragma unroll
            for (int g = 0; g < SETS; g++) ks[s][g] = *reinterpret_cast<const u4 *>(k_scales + scale_at[s] + (unsigned)(P * g * a.page));
        };
        load_keys(0);
        if constexpr (kKeysAtOnce) load_keys(1);
        auto load_value_scales = [&]() {
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int g = 0; g < SETS; g++) vs[s][g] = *reinterpret_cast<const u4 *>(v_scales + scale_at[s] + (unsigned)(P * g * a.page));
        };
        auto load_values = [&](int g) {
#pragma unroll
            for (int s = 0; s < 2; s++) load_words<VW>(vw[s][g], v_codes + at[s] + value_at + g * (P * (BITS == 4 ? 64 : 128)));
        };
        if constexpr (kAtOnce) {
            load_value_scales();
#pragma unroll
            for (int g = 0; g < SETS; g++) load_values(g);
        }
        const int tile = t * 32;
        const bool whole = tile + 32 <= lim_least && ok0 && ok1;
        ask(t + t_step);

        float y[8];
#pragma unroll
        for (int s = 0; s < 2; s++) {
            if constexpr (!kKeysAtOnce)
                if (s == 1) {
                    __builtin_amdgcn_sched_barrier(0);
                    load_keys(1);
                }
            if constexpr (P == 1) KvWords<BITS>::template part<G>(kw[s]);
            f4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int g = 0; g < SETS; g++) {
                f4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < P; i++) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(key_codes<BITS>(&kw[s][(P * g + i) * W]), q[P * g + i], d, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; r++) sum[r] = __builtin_fmaf(low_half(ks[s][g][r]), d[r], __builtin_fmaf(high_half(ks[s][g][r]), qsum[g], sum[r]));
            }
#pragma unroll
            for (int r = 0; r < 4; r++) y[4 * s + r] = cols_sum<P>(sum[r]) * key_scale;
        }
        if constexpr (!kAtOnce) {
            __builtin_amdgcn_sched_barrier(0);
            load_value_scales();
#pragma unroll
            for (int g = 0; g < kFirst; g++) load_values(g);
        }
        // (as in mha_kv_kernel; masks, since two values of every scale would take as many registers again)
        unsigned seen[8];
#pragma unroll
        for (int e = 0; e < 8; e++) seen[e] = ~0u;
        if (!whole) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int s = e >> 2, pos = tile + 16 * s + 4 * j + (e & 3);
                const bool is = (s == 0 ? ok0 : ok1) && pos < lim;
                seen[e] = is ? ~0u : 0u;
                y[e] = is ? y[e] : kNothing;
            }
        }
#pragma unroll
        for (int g = 0; g < SETS; g++)
#pragma unroll
            for (int e = 0; e < 8; e++) vs[e >> 2][g][e & 3] &= seen[e];
        // the largest scale: they are not negative, and their bits in the low halves of the words go up with them
        typedef unsigned short s2 __attribute__((ext_vector_type(2)));
        auto halves = [](unsigned w) { return __builtin_bit_cast(s2, w); };  // (of an element of a vector, __builtin_bit_cast takes the vector's first)
        auto scale_of = [&](int g) {
            s2 m = halves(vs[0][g][0]);
#pragma unroll
            for (int e = 1; e < 8; e++) m = __builtin_elementwise_max(m, halves(vs[e >> 2][g][e & 3]));
            return m;
        };
        auto exponent = [](s2 m) { return (float)__builtin_amdgcn_frexp_expf(low_half(__builtin_bit_cast(unsigned, m))); };
        s2 most_s = scale_of(0);
#pragma unroll
        for (int g = 1; g < SETS; g++) most_s = __builtin_elementwise_max(most_s, scale_of(g));
        const float most_e = exponent(most_s);
        float most_y = y[0];
#pragma unroll
        for (int e = 1; e < 8; e++) most_y = fmaxf(most_y, y[e]);
        const float reach = most_y + most_e;
        // (computed anew wherever it is used: there are no registers to keep what the compiler would like to)
        auto group_exponent = [&](int g) {
            unsigned first = vs[0][g][0];
            asm("" : "+v"(first));
            vs[0][g][0] = first;
            return exponent(scale_of(g));
        };
        const bool moves = __any(reach > ref + 15.0f);
        if (moves || lifted) {
            bool choose = false;
            if (moves) {
                float least_e = most_e;
#pragma unroll
                for (int g = 0; g < SETS; g++) least_e = fminf(least_e, group_exponent(g));
                choose = __any(most_e - least_e > kLeastLift);
                const float next = fmaxf(ref, rows_max(reach) - 11.0f);
                const float f = __builtin_amdgcn_exp2f(ref - next);
                ref = next;
                l *= f;
                float fr[4];
#pragma unroll
                for (int r = 0; r < 4; r++) fr[r] = __shfl(f, 4 * j + r);
#pragma unroll
                for (int g = 0; g < SETS; g++) {
                    z[g] *= f;
#pragma unroll
                    for (int k = 0; k < PRODUCTS; k++)
#pragma unroll
                        for (int r = 0; r < 4; r++) acc[g][k][r] *= fr[r];
                }
            }
            if (choose || lifted) {
                // the scales themselves are lifted, where times 2^lift they stay binary16 numbers
                unsigned lifts = 0;
#pragma unroll
                for (int g = 0; g < SETS; g++) {
                    const float e = group_exponent(g);
                    lifts |= (unsigned)next_lift((float)lift_of(lift, g), rows_max(most_y - ref + e), kMostLift - fmaxf(rows_max(e), 0.0f), choose) << (4 * g);
                }
                int was[4], now[4];  // of rows 4 j .. 4 j + 3 of the products
#pragma unroll
                for (int r = 0; r < 4; r++) was[r] = __shfl((int)lift, 4 * j + r), now[r] = __shfl((int)lifts, 4 * j + r);
                lift = lifts;
                lifted = __any(lift != 0);
#pragma unroll
                for (int g = 0; g < SETS; g++) {
#pragma unroll
                    for (int r = 0; r < 4; r++)
#pragma unroll
                        for (int k = 0; k < PRODUCTS; k++) acc[g][k][r] = __builtin_ldexpf(acc[g][k][r], lift_of(now[r], g) - lift_of(was[r], g));
                    const h2 m = {(_Float16)__builtin_ldexpf(1.0f, lift_of(lift, g)), (_Float16)1.0f};
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const unsigned sl = vs[e >> 2][g][e & 3];
                        vs[e >> 2][g][e & 3] = __builtin_bit_cast(unsigned, h2(__builtin_bit_cast(h2, sl) * m));
                    }
                }
            }
        }
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            p[e] = y[e] == kNothing ? 0.0f : __builtin_amdgcn_exp2f(y[e] - ref);
            l += p[e];
        }
#pragma unroll
        for (int g = 0; g < SETS; g++) {
            if (g + kFirst < SETS) {
                __builtin_amdgcn_sched_barrier(0);
                load_values(g + kFirst);
            }
            h8 w, rest;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const unsigned sl = vs[e >> 2][g][e & 3];
                _Float16 we, re;
                weight_of<true>(we, re, p[e], sl, zero);
                w[e] = we, rest[e] = re;
                z[g] = __builtin_fmaf(p[e], high_half(sl), z[g]);
            }
#pragma unroll
            for (int k = 0; k < PRODUCTS; k++) {
                unsigned x[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if constexpr (BITS == 8) x[i] = raised<8>(vw[i >> 1][g][(k >> 1) * 2 + (i & 1)], k & 1);
                    else if constexpr (P == 2) x[i] = raised<4>(vw[i >> 1][g][i & 1], k);
                    else x[i] = (k == 0 ? vw[i >> 1][g][i & 1] >> code_at << 7 : vw[i >> 1][g][i & 1] >> code_at << 3) & 0x07800780u;
                }
                const h8 codes = as_h8(x[0], x[1], x[2], x[3]);
                acc[g][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, codes, acc[g][k], 0, 0, 0);
                acc[g][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(rest, codes, acc[g][k], 0, 0, 0);
            }
        }
    }

    if (lifted) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const unsigned of_row = (unsigned)__shfl((int)lift, 4 * j + r);
#pragma unroll
            for (int g = 0; g < SETS; g++)
#pragma unroll
                for (int k = 0; k < PRODUCTS; k++) acc[g][k][r] = __builtin_ldexpf(acc[g][k][r], -lift_of(of_row, g));
        }
    }

    // what the waves have, side by side
    const float ls = rows_sum(l);
    if (j == 0) lds_stats[wave][0][c] = ref, lds_stats[wave][1][c] = ls;
#pragma unroll
    for (int g = 0; g < SETS; g++) {
        const float zs = rows_sum(z[g]);
        if (j == 0) lds_stats[wave][2 + g][c] = zs;
        const int ch = P == 2 ? g * 64 + 4 * c : g * 32 + (BITS == 4 ? 4 * (c & 7) + 2 * (c >> 3) : 2 * c);
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int k = 0; k < PRODUCTS; k++)
                if (P == 1 || (r & 1) == c >> 3) lds_vals[wave][(4 * j + r) / P * HD + ch + k] = acc[g][k][r] * (P == 1 && BITS == 4 ? 0x1p17f : code_unit<BITS>(k));
    }
    __syncthreads();
    float *part = splits > 1 ? a.parts + ((size_t)blockIdx.z * units + (unsigned)(b * nkv + kv)) * (32 + ROWS * HD) : nullptr;
    for (int e = threadIdx.x; e < rows * HD; e += NW * 64) {
        const int h = e / HD, ch = e - h * HD, g = ch >> 5, col = h * P + g % P;
        float m = lds_stats[0][0][col];
#pragma unroll
        for (int w = 1; w < NW; w++) m = fmaxf(m, lds_stats[w][0][col]);
        float sum = 0.0f, ls = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = __builtin_amdgcn_exp2f(lds_stats[w][0][col] - m);
            sum = __builtin_fmaf(f, lds_vals[w][e] + lds_stats[w][2 + g / P][col], sum);
            ls = __builtin_fmaf(f, lds_stats[w][1][col], ls);
        }
        if (part) {
            part[32 + e] = sum;
            if (g < P && (ch & 31) == 0) part[2 * col] = m, part[2 * col + 1] = ls;
        } else {
            const int row = row0 + h, i = row_of(row), r = row - i * per;
            a.Z[((size_t)b * n + i) * a.ldz + (size_t)(kv * per + r) * HD + ch] = result_value(sum, ls);
        }
    }
}

// Few rows a key/value head (R: 1, or the 4 / kCols that fill the products' rows): a tile of 64 keys whose scores end one a lane, so that the softmax costs a key once.
//
// Scores: rows of the products are the groups of the query rows, four times over, columns 16 keys; a lane keeps those of piece lane / 16 of the tile.  Group by group
// they are scaled and added in the lane.  The weights go through 1 KB of LDS (one wave's own, no barrier) to become the rows of the products with the values.
//
// Bound by memory: 64 sequences of 4096 tokens, 16 heads of 64, 4 bits 49.5 us, 5.1 TB/s (64.6 in tiles of 32 keys, whose softmax every group of a row repeats).
template <int BITS, int HD, int R> struct KvFew {
    static constexpr int kCols = KvShape<BITS, HD>::kCols;  // 1, 2 or 4 groups of a head
    static constexpr int kLdsRow = 72;                      // halfs: 64 keys, and 16 bytes on to other banks
    static constexpr int kLdsWave = 4 * kLdsRow * 2 > R * HD * 2 ? 4 * kLdsRow * 2 : R * HD * 2;  // halfs of a wave: the weights and their rests; at the end its results
    static constexpr int kPart = 32 + R * HD;
};

template <int BITS, int HD> constexpr int kv_few_waves() { return BITS == 8 && HD == 128 ? 3 : HD > 64 ? 4 : 5; }

template <int BITS, int HD, int R, int NW> __global__ __launch_bounds__(NW * 64, (kv_few_waves<BITS, HD>())) void mha_kv_few_kernel(KV_LEADING, const KvMhaArgs a) {
    using S = KvShape<BITS, HD>;
    using F = KvFew<BITS, HD, R>;
    constexpr int GP = F::kCols, G = S::kGroups, TB = S::kTokenBytes;
    __shared__ __align__(16) _Float16 lds[NW][F::kLdsWave];
    __shared__ float lds_stats[NW][R][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, j = lane >> 4;
    const int kv = blockIdx.x, b = blockIdx.y, nkv = gridDim.x;
    const int block = splits == 1 ? blockIdx.z : blockIdx.z / splits, split = blockIdx.z - block * splits;

    // Tiles are dealt to the waves of all workgroups in turn, whatever the sequence's length: the first one's pages are asked for together with it.
    const auto *table = ET_KV_CONST(int32_t, table_at) + (size_t)b * max_pages;
    const int t_step = splits * NW;
    int t = split * NW + wave;
    const bool wide = (page_pieces & 3) == 0;  // a tile lies in one page
    int page[4], off[4];
    auto ask = [&](int tile) {
        const int piece = 4 * tile;
        int pidx = (int)(((unsigned long long)(unsigned)piece * magic) >> shift), at = piece - pidx * page_pieces;
        off[0] = at << 4;
        page[0] = pidx < max_pages ? table[pidx] : -1;
        if (wide) return;
#pragma unroll
        for (int s = 1; s < 4; s++) {
            const bool on = ++at == page_pieces;
            at = on ? 0 : at;
            pidx += on;
            off[s] = at << 4;
            page[s] = pidx < max_pages ? table[pidx] : -1;
        }
    };
    ask(t);

    // the rows of this block, and what they see
    const int start = starts_at ? ET_KV_CONST(int32_t, starts_at)[b] : 0;
    const int count = counts_at ? min(max(ET_KV_CONST(int32_t, counts_at)[b], 0), n) : n;
    const int row0 = block * R, rows = min(R, count * per - row0);
    if (rows <= 0) return;
    const long long most = (long long)max_pages * a.page;
    const int end = (int)min(max((long long)start + count, 0LL), most);
    auto row_of = [&](int row) { return n == 1 ? 0 : row / per; };  // of the call's rows
    auto limit = [&](int row) { return a.causal ? (int)min((long long)end, max((long long)start + row_of(row) + 1, 0LL)) : end; };
    int lim[R];
#pragma unroll
    for (int h = 0; h < R; h++) lim[h] = limit(row0 + min(h, rows - 1));
    const int lim_least = lim[0], lim_most = lim[R - 1];
    const int t_end = (lim_most + 63) >> 6;

    // Q as in mha_kv_kernel; row c of the products is group c % GP of query row c / GP % HP
    const int h_own = (c & 3) / GP, g_own = c % GP;
    h8 q[S::kPieces];
    float key_scale[R], qsum[R][G];
    {
        const int row = row0 + min(h_own, rows - 1), i_row = row_of(row), r_row = row - i_row * per;
        const _Float16 *qrow = a.Q + ((size_t)b * n + i_row) * a.ldq + (size_t)(kv * per + r_row) * HD + j * (HD / 4);
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < S::kPieces; i++) {
            q[i] = *reinterpret_cast<const h8 *>(qrow + 8 * i);
#pragma unroll
            for (int k = 0; k < 8; k++) top = fmaxf(top, fabsf((float)q[i][k]));
        }
        top = rows_max(top);
        const int up = top > 0.0f ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
        const float grow = query_growth(top, up, a.scale_log2e);
        const float back = __builtin_ldexpf(fabsf(a.scale_log2e), key_unit_log2<BITS>() - up);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < S::kPieces; i++) q[i] = query_order<BITS>(q[i], (j * (HD / 4) + 8 * i) / 32 == g_own ? grow : 0.0f, sum);
        sum = __builtin_ldexpf(rows_sum(sum), -key_unit_log2<BITS>());
#pragma unroll
        for (int h = 0; h < R; h++) {
            key_scale[h] = lane_value(back, h * GP);
#pragma unroll
            for (int g = 0; g < G; g++) qsum[h][g] = lane_value(sum, h * GP + g);
        }
    }

    f4 acc[S::kAcc];
#pragma unroll
    for (int i = 0; i < S::kAcc; i++) acc[i] = f4{0.f, 0.f, 0.f, 0.f};
    float ref[R], l[R], z[R][G];
    unsigned lift = 0;  // of rows and groups, four bits each: what acc is times 2^ of
    auto lift_of = [](unsigned lifts, int h, int g) { return (int)(lifts >> (4 * (h * G + g)) & 15u); };
#pragma unroll
    for (int h = 0; h < R; h++) {
        ref[h] = kNothing, l[h] = 0.0f;
#pragma unroll
        for (int g = 0; g < G; g++) z[h][g] = 0.0f;
    }

    const unsigned key_at = c * TB + j * (TB / 4), value_at = j * (4 * TB) + c * (8 * S::kUnits), half_at = j * (4 * TB) + 128 * S::kUnits + (c >> 1) * 8;
    const char *k_codes = a.k_codes + (size_t)kv * a.page * TB, *v_codes = a.v_codes + (size_t)kv * a.page * TB;
    const unsigned *k_scales = a.k_scales + (size_t)kv * (G * a.page), *v_scales = a.v_scales + (size_t)kv * (G * a.page);
    const unsigned page_bytes = (unsigned)nkv * a.page * TB, page_scales = (unsigned)nkv * G * a.page;
    _Float16 *weights = lds[wave];
    // key 16 s + c of a tile among the 64 of a row: so that the keys 4 j .. 4 j + 3 of two pieces, which a lane multiplies, lie together
    const int key_place = (j >> 1) * 32 + (c >> 2) * 8 + (j & 1) * 4 + (c & 3);
    const _Float16 *weights_at = weights + (c & 3) * F::kLdsRow + j * 8;

    const float zero = hidden_zero();
    for (; t < t_end; t += t_step) {
        // where the pieces lie; one that nobody sees, or without a page, is read from the place of the one before it
        const int there = (lim_most - t * 64 + 15) >> 4;  // pieces that somebody sees, or more
        size_t at[4], scale_at;
        bool mine, all;  // this lane's piece has a page; all have
        if (wide) {
            mine = all = page[0] >= 0 && page[0] < a.npages;
            const unsigned from = mine ? page[0] : 0, from_off = mine ? off[0] : 0;
            at[0] = (size_t)from * page_bytes + from_off * TB;
#pragma unroll
            for (int s = 1; s < 4; s++) at[s] = at[0] + min(s, there - 1) * (16 * TB);
            scale_at = (size_t)from * page_scales + (from_off + lane);
        } else {
            int from = 0, from_off = 0, from_own = 0, off_own = 0;
            mine = false;
            all = true;
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const bool ok = s < there && page[s] >= 0 && page[s] < a.npages;
                from = ok ? page[s] : from;
                from_off = ok ? off[s] : from_off;
                at[s] = (size_t)(unsigned)from * page_bytes + (unsigned)from_off * TB;
                from_own = j == s ? from : from_own;
                off_own = j == s ? from_off : off_own;
                mine = j == s ? ok : mine;
                all &= ok;
            }
            scale_at = (size_t)(unsigned)from_own * page_scales + (unsigned)(off_own + c);
        }
        unsigned kw[4][S::kKeyWords], vw[4][S::kValueWords], ks[G], vs[G];
#pragma unroll
        for (int s = 0; s < 4; s++) load_words<S::kKeyWords>(kw[s], k_codes + at[s] + key_at);
#pragma unroll
        for (int g = 0; g < G; g++) ks[g] = k_scales[scale_at + (unsigned)(g * a.page)];
#pragma unroll
        for (int g = 0; g < G; g++) vs[g] = v_scales[scale_at + (unsigned)(g * a.page)];
#pragma unroll
        for (int s = 0; s < 4; s++) load_value<BITS, HD>(vw[s], v_codes + at[s] + value_at, v_codes + at[s] + half_at);
        ask(t + t_step);

        // scores: every piece's products give all lanes of a column the same; a lane keeps those of piece j
        f4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 4; s++) {
            f4 e = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < S::kPieces; i++) e = __builtin_amdgcn_mfma_f32_16x16x32_f16(q[i], key_codes<BITS>(&kw[s][i * BITS / 4]), e, 0, 0, 0);
#pragma unroll
            for (int x = 0; x < 4; x++)
                if (x < R * GP && x % GP < G) d[x] = s == 0 || j == s ? e[x] : d[x];
        }
        const int pos = t * 64 + lane;
        const bool whole = t * 64 + 64 <= lim_least && all;
        if (!whole && (pos >= lim_most || !mine)) {
#pragma unroll
            for (int g = 0; g < G; g++) vs[g] = 0;
        }
        float most_s = low_half(vs[0]);
#pragma unroll
        for (int g = 1; g < G; g++) most_s = fmaxf(most_s, low_half(vs[g]));
        const float most_e = (float)__builtin_amdgcn_frexp_expf(most_s);
#pragma unroll
        for (int h = 0; h < R; h++) {
            float y = 0.0f;
#pragma unroll
            for (int g = 0; g < G; g++) y = __builtin_fmaf(low_half(ks[g]), d[h * GP + g], __builtin_fmaf(high_half(ks[g]), qsum[h][g], y));
            y *= key_scale[h];
            const bool seen = whole || (pos < lim[h] && mine);
            y = seen ? y : kNothing;
            // a weight is at most 2^15: p * scale < 2^(y - ref + exponent of the scale)
            const float reach = y + most_e;
            const bool moves = __any(reach > ref[h] + 15.0f);
            if (moves || (G > 1 && lift != 0)) {
                bool choose = false;
                if (moves) {
                    if constexpr (G > 1) {
                        int least_e = __builtin_amdgcn_frexp_expf(low_half(vs[0]));
#pragma unroll
                        for (int g = 1; g < G; g++) least_e = min(least_e, __builtin_amdgcn_frexp_expf(low_half(vs[g])));
                        choose = __any(most_e - (float)least_e > kLeastLift);
                    }
                    const float next = fmaxf(ref[h], wave_max(reach) - 11.0f);
                    const float f = __builtin_amdgcn_exp2f(ref[h] - next);
                    ref[h] = next;
                    l[h] *= f;
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        z[h][g] *= f;
#pragma unroll
                        for (int i = 0; i < S::kAcc; i++) acc[i][h * GP + g] *= f;
                    }
                }
                if (G > 1 && (choose || lift != 0)) {
                    unsigned lifts = lift;
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        const int was = lift_of(lift, h, g), at = 4 * (h * G + g);
                        const int now = (int)next_lift((float)was, wave_max(y - ref[h] + (float)__builtin_amdgcn_frexp_expf(low_half(vs[g]))), kMostLift, choose);
                        lifts = (lifts & ~(15u << at)) | (unsigned)now << at;
#pragma unroll
                        for (int i = 0; i < S::kAcc; i++) acc[i][h * GP + g] = __builtin_ldexpf(acc[i][h * GP + g], now - was);
                    }
                    lift = __builtin_amdgcn_readfirstlane(lifts);
                }
            }
            const float p = seen ? __builtin_amdgcn_exp2f(y - ref[h]) : 0.0f;
            l[h] += p;
#pragma unroll
            for (int g = 0; g < G; g++) {
                z[h][g] = __builtin_fmaf(p, R == 1 || seen ? high_half(vs[g]) : 0.0f, z[h][g]);  // (what others see may be NaN, and 0 * NaN is)
                _Float16 w, rest;
                weight_of(w, rest, G == 1 ? p : __builtin_ldexpf(p, lift_of(lift, h, g)), vs[g], zero);
                weights[(h * GP + g) * F::kLdsRow + key_place] = w;
                weights[(4 + h * GP + g) * F::kLdsRow + key_place] = rest;
            }
        }
        wave_lds_order();
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const h8 w = *reinterpret_cast<const h8 *>(weights_at + u * 32), rest = *reinterpret_cast<const h8 *>(weights_at + 4 * F::kLdsRow + u * 32);
            weigh_values<BITS, HD>(acc, w, rest, vw[2 * u], vw[2 * u + 1], c);
        }
        wave_lds_order();
    }

    if (G > 1 && lift != 0) {
#pragma unroll
        for (int h = 0; h < R; h++)
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int i = 0; i < S::kAcc; i++) acc[i][h * GP + g] = __builtin_ldexpf(acc[i][h * GP + g], -lift_of(lift, h, g));
    }

    // what the waves have, side by side
    float *vals = reinterpret_cast<float *>(lds[wave]);
#pragma unroll
    for (int h = 0; h < R; h++) {
        const float sum = wave_sum(l[h]);
        if (lane == 0) lds_stats[wave][h][0] = ref[h], lds_stats[wave][h][1] = sum;
#pragma unroll
        for (int g = 0; g < G; g++) z[h][g] = wave_sum(z[h][g]);
    }
    // (rows 4, 5, .. of these products are rows 0, 1, .. again: the first 16 lanes store)
#pragma unroll
    for (int i = 0; i < S::kAcc; i++) {
        const int ch = value_channel<BITS, HD>(i, c);
#pragma unroll
        for (int h = 0; h < R; h++)
#pragma unroll
            for (int g = 0; g < G; g++)
                if (j == 0 && g == ch >> 5) vals[h * HD + ch] = __builtin_fmaf(acc[i][h * GP + g], value_unit<BITS, HD>(i), z[h][g]);
    }
    __syncthreads();
    float *part = splits > 1 ? a.parts + ((size_t)blockIdx.z * units + (unsigned)(b * nkv + kv)) * F::kPart : nullptr;
    for (int e = threadIdx.x; e < rows * HD; e += NW * 64) {
        const int h = e / HD, ch = e - h * HD;
        float m = lds_stats[0][h][0];
#pragma unroll
        for (int w = 1; w < NW; w++) m = fmaxf(m, lds_stats[w][h][0]);
        float sum = 0.0f, ls = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = __builtin_amdgcn_exp2f(lds_stats[w][h][0] - m);
            sum = __builtin_fmaf(f, reinterpret_cast<const float *>(lds[w])[e], sum);
            ls = __builtin_fmaf(f, lds_stats[w][h][1], ls);
        }
        if (part) {
            part[32 + e] = sum;
            if ((ch & 31) == 0) part[2 * (h * GP + (ch >> 5))] = m, part[2 * (h * GP + (ch >> 5)) + 1] = ls;
        } else {
            const int row = row0 + h, i = row_of(row), r = row - i * per;
            a.Z[((size_t)b * n + i) * a.ldz + (size_t)(kv * per + r) * HD + ch] = result_value(sum, ls);
        }
    }
}

// The parts of a unit's rows: 32 threads a channel group of a row, or 2, 4, 8 times that many where there are many parts, which a workgroup then adds up (lots: how many).
// (One workgroup of eight for each, whatever the parts, was 8192 waves to start for 16 sequences of 32 heads over 8 of 128, 4096 tokens in four parts: 24.0 us with
// the attention, 22.9 so.)
__global__ __launch_bounds__(256) void mha_kv_join_kernel(const KvMhaArgs a, int lots_log2) {
    __shared__ float lds[3][8][32];
    const int groups = a.hd / ET_KV_GROUP, part_floats = 32 + a.block_rows * a.hd, lots = 1 << lots_log2;
    const int ch = threadIdx.x & 31, at_once = threadIdx.x >> 5, lot = at_once & (lots - 1);
    const int mine = (int)blockIdx.x * (8 >> lots_log2) + (at_once >> lots_log2);
    const int block = blockIdx.y, unit = mine / (a.block_rows * groups), col_g = mine - unit * (a.block_rows * groups);
    const int h = col_g / groups, g = col_g - h * groups;
    const int b = unit / a.nkv, kv = unit - b * a.nkv;
    const int row = block * a.block_rows + h;
    const bool there = unit < a.units && row < (a.counts ? min(max(a.counts[b], 0), a.n) : a.n) * a.per;
    float m = kNothing, sum = 0.0f, ls = 0.0f;
    if (there) {
        const float *part = a.parts + ((size_t)block * a.splits * a.units + unit) * part_floats;
        const size_t next = (size_t)a.units * part_floats;
        const int col = h * a.cols + (g & (a.cols - 1)), at = 32 + h * a.hd + g * 32 + ch;
        for (int s0 = lot; s0 < a.splits; s0 += 4 * lots) {  // four parts asked for at once
            float pm[4], pl[4], pv[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const bool is = s0 + k * lots < a.splits;
                const float *p = part + (is ? s0 + k * lots : s0) * next;
                pm[k] = is ? p[2 * col] : kNothing;
                pl[k] = is ? p[2 * col + 1] : 0.0f;
                pv[k] = is ? p[at] : 0.0f;
            }
            const float most = fmaxf(fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])), m);
            const float f = __builtin_amdgcn_exp2f(m - most);
            m = most;
            sum *= f;
            ls *= f;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float fk = __builtin_amdgcn_exp2f(pm[k] - most);
                sum = __builtin_fmaf(fk, pv[k], sum);
                ls = __builtin_fmaf(fk, pl[k], ls);
            }
        }
    }
    if (lots > 1) {
        lds[0][at_once][ch] = m, lds[1][at_once][ch] = sum, lds[2][at_once][ch] = ls;
        __syncthreads();
        if (lot != 0) return;
        for (int w = at_once + 1; w < at_once + lots; w++) {
            const float mw = lds[0][w][ch], most = fmaxf(m, mw), f = __builtin_amdgcn_exp2f(m - most), fw = __builtin_amdgcn_exp2f(mw - most);
            m = most;
            sum = sum * f + lds[1][w][ch] * fw;
            ls = ls * f + lds[2][w][ch] * fw;
        }
    }
    if (!there) return;
    const int i = row / a.per, r = row - i * a.per;
    a.Z[((size_t)b * a.n + i) * a.ldz + (size_t)(kv * a.per + r) * a.hd + g * 32 + ch] = result_value(sum, ls);
}

namespace {

using KvKernel = void (*)(KV_LEADING, const KvMhaArgs);

struct KvForm {
    KvKernel four, eight;  // waves
    int rows, cols, tile;
    bool eight_if_whole;   // eight only where one workgroup has all the keys
};

// Rows: of a key/value head in the call.  fills: one block of rows for each (sequence, key/value head) is enough work for the chip, there being many, or keys to share out.
// Blocks of 16 / kCols rows or of 16, us, 8 heads, 16 sequences of 4096 tokens with heads up to 128 and 4 with wider ones, 4 bits (8 bits):
//    64: 8 rows 18.5 | 21.7 (20.1 | 21.8)   9 rows 26.6 | 21.9 (28.2 | 22.2)      96: 5 rows 30.6 | 29.7 (38.6 | 30.2)   8 rows 30.8 | 30.4 (38.8 | 31.0)   9 rows 42.5 | 30.6 (53.4 | 31.3)
//   160: 4 rows 16.7 | 17.7 (19.3 | 18.9)   5 rows 27.6 | 18.1 (31.3 | 19.0)     192: 4 rows 18.7 | 20.1 (20.4 | 20.7)   5 rows 30.8 | 20.3 (34.1 | 20.9)
//   224: 4 rows 20.0 | 23.0 (22.3 | 24.1)   5 rows 33.2 | 23.4 (37.1 | 24.3)     256: 4 rows 21.1 | 25.3 (27.8 | 26.3)   5 rows 35.1 | 25.5 (47.2 | 26.5)
// So 5 to 8 rows of heads of 96 in 8 bits are on the slower side.  Heads of 128, 5 to 8 rows: blocks of 4, of 8 over pairs of groups or of 16, us, 8 rows:
//   16 x 4096 35.0 | 31.1 | 38.5 (50.4 | 34.4 | 40.5)   16 x 2112 23.6 | 19.1 | 23.3 (30.2 | 20.3 | 24.3)   16 x 1984 19.6 | 21.9 | 27.3 (23.7 | 23.4 | 28.9)   40 x 1000 28.5 | 26.4 | 32.3 (36.1 | 27.9 | 33.4)
//   4 x 2112 14.2 | 15.7 | 15.9 (16.9 | 16.7 | 16.3)    4 x 1984 16.3 | 19.2 | 24.6 (20.8 | 21.2 | 25.9)    1 x 8000 15.5 | 17.3 | 16.1 (18.6 | 18.4 | 16.5)
// so from 2048 positions on a few sequences in 4 bits are up to 12 % on the slower side.  Wider heads: pairs are no better than 16 rows.
template <int BITS, int HD> KvForm form_of(long long rows, bool fills) {
    if constexpr (HD <= 128) {
        constexpr int cols = KvShape<BITS, HD>::kCols, heads = 4 / cols;
        if (rows == 1) return {mha_kv_few_kernel<BITS, HD, 1, 4>, mha_kv_few_kernel<BITS, HD, 1, 8>, 1, cols, 64, false};
        if (rows <= heads) return {mha_kv_few_kernel<BITS, HD, heads, 4>, mha_kv_few_kernel<BITS, HD, heads, 8>, heads, cols, 64, false};
    }
    if constexpr (HD > 32)
        if (rows > (HD <= 128 ? 8 : 4)) return {mha_kv_rows_kernel<BITS, HD, 4, 1>, mha_kv_rows_kernel<BITS, HD, HD <= 128 ? 8 : 4, 1>, 16, 1, 32, HD > 64};
    if constexpr (HD == 128)
        if (rows > 4 && fills) return {mha_kv_rows_kernel<BITS, HD, 4, 2>, mha_kv_rows_kernel<BITS, HD, 8, 2>, 8, 2, 32, false};
    return {mha_kv_kernel<BITS, HD, 4>, mha_kv_kernel<BITS, HD, 8>, KvShape<BITS, HD>::kRows, KvShape<BITS, HD>::kCols, 32, false};
}

template <int BITS> KvForm form_of(int hd, long long rows, bool fills) {
    switch (hd) {
        case 32: return form_of<BITS, 32>(rows, fills);
        case 64: return form_of<BITS, 64>(rows, fills);
        case 96: return form_of<BITS, 96>(rows, fills);
        case 128: return form_of<BITS, 128>(rows, fills);
        case 160: return form_of<BITS, 160>(rows, fills);
        case 192: return form_of<BITS, 192>(rows, fills);
        case 224: return form_of<BITS, 224>(rows, fills);
        default: return form_of<BITS, 256>(rows, fills);
    }
}

struct KvPlan {
    KvForm form;
    int blocks, splits, waves;
    size_t bytes;
};

// Waves of a workgroup and workgroups that share the keys of a (sequence, key/value head): 4096 waves, which fill the chip, but at least four tiles a wave if every
// sequence were as long as its table; a second launch, which joins the parts, costs 3 to 6 us.  Eight waves a workgroup where there are few: 16 rows, 8 heads of 128, 1000
// tokens, 32 sequences 25.1 us with four, 19.9 with eight (16 sequences 17.0 and 17.7), one row, 8 x 2048, 12 heads of 64 9.8 and 8.2; but only two of them a SIMD fit of 16 rows of
// heads of 96 and 128 (of 96 three with four waves): where keys are shared out anyway, four (16 x 10937 tokens, 5 heads of 96, 80 rows 170 and 204 us, 64 x 1000, 16 heads of 128 59 and 73).
int kv_plan(const char *fn, KvPlan &p, const et_kv_cache *c, int max_pages, int B, int n, int nh) {
    ET_REQUIRE(nh > 0 && nh % c->nkv == 0, ET_ERR_INVALID_ARG, "%s: nh=%d must be a multiple of nkv=%d", fn, nh, c->nkv);
    const int per = nh / c->nkv;
    const long long rows = (long long)n * per;
    const long long units = (long long)B * c->nkv;
    // (in tiles, which the shares below count too: were the two rounded differently, the form of fewer rows a block could need more for the last pages under the border)
    const bool fills = units >= 256 || ((long long)max_pages * c->page + 31) / 32 >= 64;
    p.form = c->bits == 4 ? form_of<4>(c->hd, rows, fills) : form_of<8>(c->hd, rows, fills);
    const long long blocks = (rows + p.form.rows - 1) / p.form.rows;
    ET_REQUIRE(rows <= 0x7fffffffLL && B <= 65535 && blocks <= 65535 && units * blocks <= (1LL << 24), ET_ERR_UNSUPPORTED, "%s: B=%d n=%d nh=%d", fn, B, n, nh);
    p.blocks = (int)blocks;
    const long long tiles = ((long long)max_pages * c->page + p.form.tile - 1) / p.form.tile, groups = units * blocks;
    p.waves = groups >= 512 || p.form.four == p.form.eight || (p.form.eight_if_whole && tiles >= 64) ? 4 : 8;
    p.splits = groups == 0 ? 1 : (int)std::max(1LL, std::min({(4096 / p.waves + groups - 1) / groups, tiles / (4 * p.waves), 256LL}));
    p.splits = std::min(p.splits, (int)(65535 / std::max(1LL, blocks)));
    p.bytes = p.splits > 1 ? (size_t)(groups * p.splits) * (32 + p.form.rows * c->hd) * sizeof(float) : 0;
    return ET_OK;
}

}  // namespace

}  // namespace et

using namespace et;

extern "C" {

int et_mha_kv_workspace(const et_kv_cache *cache, int max_pages, int B, int n, int nh, size_t *bytes) {
    ET_REQUIRE(bytes, ET_ERR_INVALID_ARG, "et_mha_kv_workspace: NULL pointer");
    static const int32_t any = 0;
    const int st = kv_check_cache("et_mha_kv_workspace", cache, &any, max_pages, B, n);
    if (st != ET_OK) return st;
    KvPlan p;
    const int sp = kv_plan("et_mha_kv_workspace", p, cache, max_pages, B, n, nh);
    if (sp == ET_OK) *bytes = p.bytes;
    return sp;
}

int et_mha_kv_f16(const et_kv_cache *cache, const int32_t *table, int max_pages, const int32_t *starts, const int32_t *counts, const et_f16 *Q, int ldq,
                  et_f16 *Z, int ldz, int B, int n, int nh, float scale, int flags, void *workspace, size_t workspace_bytes, et_stream stream) {
    ET_REQUIRE(Q && Z, ET_ERR_INVALID_ARG, "et_mha_kv_f16: NULL pointer");
    const int st = kv_check_cache("et_mha_kv_f16", cache, table, max_pages, B, n);
    if (st != ET_OK) return st;
    ET_REQUIRE((flags & ~ET_MHA_CAUSAL) == 0, ET_ERR_INVALID_ARG, "et_mha_kv_f16: flags=%d", flags);
    // (scores stay below 1e30 in magnitude, which stands for minus infinity; 256 products of binary16 numbers reach 1.1e12)
    ET_REQUIRE(fabsf(scale) <= 1e15f, ET_ERR_INVALID_ARG, "et_mha_kv_f16: scale=%g", (double)scale);
    KvPlan p;
    const int sp = kv_plan("et_mha_kv_f16", p, cache, max_pages, B, n, nh);
    if (sp != ET_OK) return sp;
    const long long width = (long long)nh * cache->hd;
    ET_REQUIRE(ldq >= width && ldz >= width, ET_ERR_INVALID_ARG, "et_mha_kv_f16: row strides %d, %d below nh * hd = %lld", ldq, ldz, width);
    ET_REQUIRE(ldq % 8 == 0 && ldz % 8 == 0, ET_ERR_UNSUPPORTED, "et_mha_kv_f16: row strides must be multiples of 8");
    ET_REQUIRE(((reinterpret_cast<uintptr_t>(Q) | reinterpret_cast<uintptr_t>(Z)) & 15) == 0, ET_ERR_UNSUPPORTED,
               "et_mha_kv_f16: Q and Z must be 16-byte aligned");
    ET_REQUIRE(workspace_bytes >= p.bytes && (workspace || p.bytes == 0), ET_ERR_INVALID_ARG, "et_mha_kv_f16: a workspace of %zu bytes, %zu are needed",
               workspace ? workspace_bytes : 0, p.bytes);
    ET_REQUIRE(p.bytes == 0 || (reinterpret_cast<uintptr_t>(workspace) & 15) == 0, ET_ERR_UNSUPPORTED, "et_mha_kv_f16: the workspace must be 16-byte aligned");
    if (B == 0 || n == 0) return ET_OK;
    KvMhaArgs a;
    a.k_codes = static_cast<const char *>(cache->k_codes);
    a.v_codes = static_cast<const char *>(cache->v_codes);
    a.k_scales = reinterpret_cast<const unsigned *>(cache->k_scales);
    a.v_scales = reinterpret_cast<const unsigned *>(cache->v_scales);
    a.counts = counts;
    a.Q = reinterpret_cast<const _Float16 *>(Q);
    a.Z = reinterpret_cast<_Float16 *>(Z);
    a.parts = static_cast<float *>(workspace);
    a.ldq = ldq;
    a.ldz = ldz;
    a.nkv = cache->nkv;
    a.per = nh / cache->nkv;
    a.page = cache->page;
    a.npages = cache->npages;
    a.n = n;
    a.causal = flags & ET_MHA_CAUSAL;
    a.hd = cache->hd;
    a.cols = p.form.cols;
    a.block_rows = p.form.rows;
    a.units = B * cache->nkv;
    a.splits = p.splits;
    // pieces below 2^27 (and a few tiles on): piece / d = piece * ceil(2^s / d) >> s with s = 28 + ceil(log2 d)
    const unsigned d = (unsigned)cache->page / 16;
    unsigned shift = 28;
    while ((1ull << (shift - 28)) < d) shift++;
    const unsigned magic = (unsigned)(((1ull << shift) + d - 1) / d);
    a.scale_log2e = scale * 1.4426950408889634f;
    const int sl = launch_kernel("mha_kv_kernel", p.waves == 4 ? p.form.four : p.form.eight, dim3((unsigned)cache->nkv, (unsigned)B, (unsigned)(p.blocks * p.splits)), p.waves * 64, 0, as_stream(stream),
                                 table, starts, counts, max_pages, a.units, a.splits, a.per, magic, shift, (int)d, n, a);
    if (sl != ET_OK || p.splits == 1) return sl;
    const int lots_log2 = p.splits <= 4 ? 0 : p.splits <= 8 ? 1 : p.splits <= 16 ? 2 : 3;
    const int channels = a.units * p.form.rows * (cache->hd / ET_KV_GROUP), of_workgroup = 8 >> lots_log2;
    return launch_kernel("mha_kv_join_kernel", mha_kv_join_kernel, dim3((unsigned)((channels + of_workgroup - 1) / of_workgroup), (unsigned)p.blocks), 256, 0, as_stream(stream), a,
                         lots_log2);
}

}  // extern "C"
