// Linear with 4-bit weights, a scale and a lowest value for every 32, 64 or 128 input features of an output feature (layout: et_abi.h).
#include <atomic>

#include "group_quant.hip.h"

namespace et {

template <int GROUP> __global__ __launch_bounds__(256) void dense_to_w4_kernel(const _Float16 *W, unsigned *codes, unsigned *scales, int in, int out, unsigned total) {
    // a lane holds eight values; GROUP / 8 neighbouring lanes (4, 8 or 16) a group
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    if (i >= total) return;  // (total is a multiple of GROUP / 8, and so are a wave's first and last)
    const h8 x = reinterpret_cast<const h8 *>(W)[i];
    unsigned magnitude, tiny, word[1], scale_low;
    h2 e = extremes(x, magnitude, tiny);
    extremes_across<kDppQuadXor1>(e, magnitude);
    extremes_across<kDppQuadXor2>(e, magnitude);
    if constexpr (GROUP >= 64) extremes_across<0x141>(e, magnitude);          // row_half_mirror: the other four of eight
    if constexpr (GROUP >= 128) extremes_across<kDppRowRor8>(e, magnitude);
    const h8 all[1] = {x};
    quantise<4, 1>(word, scale_low, all, e, magnitude, tiny);
    codes[i] = word[0];
    const unsigned per_row = (unsigned)in / 8, o = i / per_row, at = i - o * per_row;
    if (at % (GROUP / 8) == 0) scales[(size_t)(at / (GROUP / 8)) * out + o] = scale_low;
}

__global__ __launch_bounds__(256) void w4_to_dense_kernel(const unsigned *codes, const unsigned *scales, _Float16 *W, int in, int out, int group, unsigned total) {
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    if (i >= total) return;
    const unsigned per_row = (unsigned)in / 8, o = i / per_row, at = i - o * per_row;
    const unsigned sl = scales[(size_t)(at * 8 / (unsigned)group) * out + o], word = codes[i];
    const float s = f16_bits_value(sl & 0xffffu), lo = f16_bits_value(sl >> 16);
    h8 x;
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] = step_value((float)(word >> (4 * k) & 15u), lo, s);
    reinterpret_cast<h8 *>(W)[i] = x;
}

struct W4Args {
    const unsigned char *codes;
    const unsigned *scales;  // scale in the low half, low in the high one
    const _Float16 *bias, *X;
    _Float16 *Y;
    float *Y32;
    int T, in, out, act;
};

typedef unsigned w4u __attribute__((ext_vector_type(4)));

constexpr int kW4Raw = 0x00020000;             // word 3 of a resource: raw, 32-bit data
constexpr unsigned kW4Nothing = 0x80000000u;  // an offset behind every resource: reads as zero

__device__ __forceinline__ w4u w4_load(__amdgpu_buffer_rsrc_t r, unsigned lane_at, int at) {
    return __builtin_bit_cast(w4u, __builtin_amdgcn_raw_buffer_load_b128(r, (int)lane_at, at, 0));
}

__device__ __forceinline__ h8 w4_h8(unsigned a, unsigned b, unsigned c, unsigned d) { return __builtin_bit_cast(h8, w4u{a, b, c, d}); }

// The eight codes of a word as binary16 numbers, code * 2^-17 (bits 7 to 10: up to 7 subnormal, as far apart from 8 on), in the order 0 4 1 5 2 6 3 7.
__device__ __forceinline__ h8 w4_codes(unsigned w) {
    constexpr unsigned m = 0x07800780u;
    return w4_h8((w << 7) & m, (w << 3) & m, (w >> 1) & m, (w >> 5) & m);
}
// Eight activations in the same order.
__device__ __forceinline__ h8 w4_order(w4u x) {
    constexpr unsigned lows = 0x05040100u, highs = 0x07060302u;
    return w4_h8(__builtin_amdgcn_perm(x[2], x[0], lows), __builtin_amdgcn_perm(x[2], x[0], highs), __builtin_amdgcn_perm(x[3], x[1], lows),
                 __builtin_amdgcn_perm(x[3], x[1], highs));
}

__device__ __forceinline__ float w4_scale(unsigned sl) { return (float)__builtin_bit_cast(h2, sl)[0]; }
__device__ __forceinline__ float w4_low(unsigned sl) { return (float)__builtin_bit_cast(h2, sl)[1]; }

// Y = act(X W^T + bias), W = low + scale * code.  Rows of the products are 16 output features, contraction is over the codes as they are, 128 input features ("a chunk") in
// four products; scale and low come to a group's binary32 sums: y += scale * sum x code + low * sum x, the second sum from products with ones.
//   SWAP 0: a lane's 16 bytes of a weight row are 32 input features, so the four lanes of a row hold the groups of a chunk side by side.  The products' columns are (row of
//           X, group), zero outside the group: 16 / groups rows of X at a time.  GROUP 128: 16 rows.
//   SWAP 1 (groups of 32 and 64, more rows): four (two) row swaps bring the words of one group into one register; columns are 16 rows of X.
// A wave has RBK blocks of 16 output features, TBK blocks of columns of which TR rows of X are real, and takes U chunks at a time.  What it loads, 64 U bytes of a weight row and 256 U of X in a
// piece, goes through LDS of its own to the lanes that multiply it: asked for by those, every 16 bytes were an access of the vector cache of their own, 52 an instruction, which bound
// the kernel at 2.2 TB/s (16 rows, 8192 to 28672 features).  The next U chunks are in flight meanwhile.  The four or eight waves of a workgroup share the chunks of its
// blocks and add up through LDS.
//
// 8192 to 28672 features in groups of 128, 126 MB: 1 row 28.4 us (4.4 TB/s), 16 rows 33 (3.8; evening out the workgroups over the compute units changes nothing).  45 rows, 4096 to 4096 in groups of 32: 11 us, every compute unit takes in all of X, 368 KB, and passes it through LDS.
template <int GROUP, int SWAP, int TBK, int TR, int RBK, int U> struct W4Shape {
    static constexpr int NG = 128 / GROUP, COLS = SWAP ? 1 : NG, TPB = 16 / COLS;  // groups of a chunk; columns of a row of X; rows of X of a column block
    static constexpr int SG = SWAP ? NG : 1;                                       // groups that a lane scales by itself
    static constexpr int kWRow = 64 * U + 16, kXRow = 256 * U + 16;                // bytes of a row in LDS: the 16 lanes of a read on different banks
    static constexpr int kW = RBK * 16 * kWRow, kX = TR * kXRow, kS = RBK * U * NG * 64;
    static constexpr int kZero = 64;
    static constexpr int kWave = kW + kX + kS + kZero;            // bytes of a wave
    static constexpr int kSum = RBK * TBK * TPB * 4 * 16;         // what it leaves in the end, in the same place
    static constexpr int kLds = kWave > kSum ? kWave : kSum;
    static constexpr int kXLoads = (TR * U * 16 + 63) / 64, kSLoads = (RBK * U * NG * 4 + 63) / 64;
};

template <int GROUP, int SWAP, int TBK, int TR, int RBK, int U> __global__ __launch_bounds__(512) void w4_linear_kernel(const W4Args a) {
    using S = W4Shape<GROUP, SWAP, TBK, TR, RBK, U>;
    constexpr int NG = S::NG, COLS = S::COLS, TPB = S::TPB, SG = S::SG;
    extern __shared__ __align__(16) char lds_all[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, j = lane >> 4;
    const int gg = c % COLS, tl = c / COLS;
    const int nb = a.out >> 4, nc = (a.in + 127) >> 7;
    const int rb0 = blockIdx.x * RBK, waves_log2 = blockDim.x == 512 ? 3 : 2;
    const int t0 = blockIdx.y * (TPB * TBK);
    char *lds_w = lds_all + wave * S::kLds, *lds_x = lds_w + S::kW, *lds_s = lds_x + S::kX, *lds_zero = lds_s + S::kS;

    // what this lane loads: pieces of 16 bytes of rows of weights, of X, of scales
    __amdgpu_buffer_rsrc_t w[RBK];
#pragma unroll
    for (int i = 0; i < RBK; i++)
        w[i] = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>(a.codes) + (size_t)(min(rb0 + i, nb - 1) * 16) * (a.in / 2), 0, 8 * a.in, kW4Raw);
    const int x_rows = min(a.T - t0, TPB * TBK);
    const auto xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<_Float16 *>(a.X) + (size_t)t0 * a.in, 0, x_rows * a.in * 2, kW4Raw);
    w4u gw[RBK][U], gx[S::kXLoads], gs[S::kSLoads];
    const int share = (nc + (1 << waves_log2) - 1) >> waves_log2, k_first = wave * share, in_end = min(a.in, (k_first + share) * 128);
    auto load = [&](int k0) {
        const int left = in_end - k0 * 128;  // input features from here on
#pragma unroll
        for (int i = 0; i < U; i++) {
            const int row = (i * 64 + lane) / (4 * U), piece = lane % (4 * U);
            const unsigned at = 32 * piece < left ? row * (a.in / 2) + 16 * piece : kW4Nothing;
#pragma unroll
            for (int r = 0; r < RBK; r++) gw[r][i] = w4_load(w[r], at, k0 * 64);
        }
#pragma unroll
        for (int i = 0; i < S::kXLoads; i++) {
            const int row = (i * 64 + lane) / (16 * U), piece = lane % (16 * U);
            gx[i] = w4_load(xr, 8 * piece < left && row < x_rows ? row * a.in * 2 + 16 * piece : kW4Nothing, k0 * 256);
        }
#pragma unroll
        for (int i = 0; i < S::kSLoads; i++) {
            const int e = i * 64 + lane, quarter = e & 3, ug = (e >> 2) % (U * NG), r = min((e >> 2) / (U * NG), RBK - 1);
            const int grp = min(k0 * NG + ug, a.in / GROUP - 1);
            gs[i] = *reinterpret_cast<const w4u *>(a.scales + (size_t)grp * a.out + min(rb0 + r, nb - 1) * 16 + 4 * quarter);
        }
    };
    auto keep = [&]() {
#pragma unroll
        for (int i = 0; i < U; i++) {
            const int row = (i * 64 + lane) / (4 * U), piece = lane % (4 * U);
#pragma unroll
            for (int r = 0; r < RBK; r++) *reinterpret_cast<w4u *>(lds_w + (r * 16 + row) * S::kWRow + piece * 16) = gw[r][i];
        }
#pragma unroll
        for (int i = 0; i < S::kXLoads; i++) {
            const int row = (i * 64 + lane) / (16 * U), piece = lane % (16 * U);
            if (S::kXLoads * 64 == TR * U * 16 || row < TR) *reinterpret_cast<h8 *>(lds_x + row * S::kXRow + piece * 16) = w4_order(gx[i]);
        }
#pragma unroll
        for (int i = 0; i < S::kSLoads; i++)
            if (S::kSLoads * 64 == RBK * U * NG * 4 || i * 64 + lane < RBK * U * NG * 4) *reinterpret_cast<w4u *>(lds_s + (i * 64 + lane) * 16) = gs[i];
    };

    // what this lane multiplies: nothing in a column of another group, or of a row of X that is none
    const char *w_from = lds_w + c * S::kWRow + 16 * j, *s_from = lds_s + (SWAP ? 0 : gg * 64) + 16 * j;
    const char *x_from[TBK];
    int x_step[TBK];  // of a chunk
#pragma unroll
    for (int b = 0; b < TBK; b++) {
        const int t = b * TPB + tl;
        const bool mine = t < TR && (SWAP || gg == j * 32 / GROUP);
        x_from[b] = mine ? lds_x + t * S::kXRow + (!SWAP ? 64 * j : GROUP == 32 ? 16 * j : 64 * (j & 1) + 16 * (j >> 1)) : lds_zero;
        x_step[b] = mine ? 1 : 0;
    }
    if (lane < 4) *reinterpret_cast<w4u *>(lds_zero + lane * 16) = w4u{0, 0, 0, 0};

    f4 acc[RBK][TBK];
#pragma unroll
    for (int i = 0; i < RBK; i++)
#pragma unroll
        for (int b = 0; b < TBK; b++) acc[i][b] = f4{0.f, 0.f, 0.f, 0.f};

    if (k_first * 128 < in_end) load(k_first);
    for (int k0 = k_first; k0 * 128 < in_end; k0 += U) {
        wave_lds_order();
        keep();
        wave_lds_order();
        if ((k0 + U) * 128 < in_end) load(k0 + U);
#pragma unroll
        for (int u = 0; u < U; u++) {
            h8 xo[TBK][4];
            f4 sums[TBK][SG];  // of X, * 2^-17
            const h8 ones = w4_h8(0x00800080u, 0x00800080u, 0x00800080u, 0x00800080u);
#pragma unroll
            for (int b = 0; b < TBK; b++) {
#pragma unroll
                for (int g = 0; g < SG; g++) sums[b][g] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int g = !SWAP ? 0 : GROUP == 32 ? r : r & 1;
                    // the piece of a chunk that product r multiplies; the others' lanes stay at the zeros
                    const int piece = !SWAP ? 16 * r : GROUP == 32 ? 64 * r : 128 * (r & 1) + 32 * (r >> 1);
                    xo[b][r] = *reinterpret_cast<const h8 *>(x_from[b] + x_step[b] * (256 * u + piece));
                    sums[b][g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, xo[b][r], sums[b][g], 0, 0, 0);
                }
            }
#pragma unroll
            for (int i = 0; i < RBK; i++) {
                const w4u raw = *reinterpret_cast<const w4u *>(w_from + i * 16 * S::kWRow + 64 * u);
                unsigned v[4] = {raw[0], raw[1], raw[2], raw[3]};
                if constexpr (SWAP) {
                    auto swap32 = [](unsigned &p, unsigned &q) {
                        auto r = __builtin_amdgcn_permlane32_swap(p, q, false, false);
                        p = r[0], q = r[1];
                    };
                    auto swap16 = [](unsigned &p, unsigned &q) {
                        auto r = __builtin_amdgcn_permlane16_swap(p, q, false, false);
                        p = r[0], q = r[1];
                    };
                    if constexpr (GROUP == 32) {
                        swap32(v[0], v[2]);
                        swap32(v[1], v[3]);
                        swap16(v[0], v[1]);
                        swap16(v[2], v[3]);
                    } else {
                        swap32(v[0], v[1]);
                        swap32(v[2], v[3]);
                    }
                }
                h8 cd[4];
#pragma unroll
                for (int r = 0; r < 4; r++) cd[r] = w4_codes(v[r]);
                w4u sl[SG];
#pragma unroll
                for (int g = 0; g < SG; g++) sl[g] = *reinterpret_cast<const w4u *>(s_from + ((i * U + u) * NG + g) * 64);
#pragma unroll
                for (int b = 0; b < TBK; b++) {
                    f4 d[SG];
#pragma unroll
                    for (int g = 0; g < SG; g++) d[g] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int g = !SWAP ? 0 : GROUP == 32 ? r : r & 1;
                        d[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(cd[r], xo[b][r], d[g], 0, 0, 0);
                    }
#pragma unroll
                    for (int g = 0; g < SG; g++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            acc[i][b][e] = __builtin_fmaf(w4_scale(sl[g][e]), d[g][e], __builtin_fmaf(w4_low(sl[g][e]), sums[b][g][0], acc[i][b][e]));
                }
            }
        }
    }

    // a row of X over its columns, then over the waves
#pragma unroll
    for (int i = 0; i < RBK; i++)
#pragma unroll
        for (int b = 0; b < TBK; b++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if constexpr (COLS >= 2) acc[i][b][e] += dpp_move<kDppQuadXor1>(acc[i][b][e]);
                if constexpr (COLS >= 4) acc[i][b][e] += dpp_move<kDppQuadXor2>(acc[i][b][e]);
            }
    auto store = [&](int i, int b, int t_in, int quarter, f4 y) {  // four output features of a row of X
        const int t = t0 + b * TPB + t_in, o = (rb0 + i) * 16 + 4 * quarter;
        if (t >= a.T || rb0 + i >= nb) return;
        h4 bias = {0, 0, 0, 0};
        if (a.bias) bias = *reinterpret_cast<const h4 *>(a.bias + o);
        h4 out16;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            y[e] = apply_act(__builtin_fmaf(y[e], 0x1p17f, (float)bias[e]), a.act);
            out16[e] = (_Float16)y[e];
        }
        if (a.Y) *reinterpret_cast<h4 *>(a.Y + (size_t)t * a.out + o) = out16;
        else *reinterpret_cast<f4 *>(a.Y32 + (size_t)t * a.out + o) = y;
    };
    wave_lds_order();
    if (gg == 0) {
#pragma unroll
        for (int i = 0; i < RBK; i++)
#pragma unroll
            for (int b = 0; b < TBK; b++) reinterpret_cast<f4 *>(lds_w)[(i * TBK + b) * (TPB * 4) + tl * 4 + j] = acc[i][b];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < RBK * TBK * TPB * 4; e += blockDim.x) {
        const int ib = e / (TPB * 4), q = e - ib * (TPB * 4);
        auto of = [&](int w) { return reinterpret_cast<const f4 *>(lds_all + w * S::kLds)[e]; };
        f4 y = (of(0) + of(1)) + (of(2) + of(3));
        if (waves_log2 == 3) y += (of(4) + of(5)) + (of(6) + of(7));
        store(ib / TBK, ib % TBK, q >> 2, q & 3, y);
    }
}

namespace {

struct W4Form {
    void (*kernel)(W4Args);
    int rows_x, blocks, kw, lds;             // rows of X and blocks of output features of a workgroup; its waves; bytes of LDS
    std::atomic<unsigned long long> *large;  // devices where the kernel may have that much, a bit each
};

template <int GROUP, int SWAP, int TBK, int TR, int RBK, int U> W4Form w4_form_of(int kw) {
    using S = W4Shape<GROUP, SWAP, TBK, TR, RBK, U>;
    static std::atomic<unsigned long long> large{0};
    return {w4_linear_kernel<GROUP, SWAP, TBK, TR, RBK, U>, S::TPB * TBK, RBK, kw, S::kLds * kw, &large};
}

// Blocks of output features (nb of them) a wave, and waves that share a block: fewer blocks fill the chip, more of them take what is loaded and ordered of X further.
// Measured, in us (nb 256 is 1024 -> 4096 and 4096 -> 4096, 512 is 4096 -> 8192, 1024 is 8192 -> 16384 and 4096 -> 16384, 1792 is 8192 -> 28672, 1800 is 800 -> 28800), for
// 1 block of eight waves, and 1, 2 and 4 blocks of four:
//   1 row             nb 256: 3.8 3.5 3.8  -    nb 1800: 10.9 6.9 6.1  -
//   16 rows, 128s     nb 1024:  -  21.6 18.0 19.5   nb 1792: 55 44.9 36.5 33.5
//   16 rows, 32s      nb 512:  9.6  -  10.6 13.3    nb 1024: 16.1  -  13.3 14.5   nb 1792: 54.8  -  44.6 40.1
//   32 rows, 32s      nb 256:  9.1 11.0 12.1  -     nb 512: 15.4  -  13.3 17.6
//   32 rows, 128s     nb 1792:  76  71  53.6 42.3
//   45 rows, 32s      nb 256: 11.5 12.8 15.8  -     nb 1792: 116 105 83  -
//   64 rows, 32s      nb 256: 15.3 13.6 12.5 17.9   nb 512: 27.9  -  18.2 18.4    nb 1792:  -   -  105  99
//   256 rows, 128s    nb 256: 42.7 33.1 23.3 19.7   nb 1792: 500 448 304 243
template <int GROUP> W4Form w4_form(int T, int nb) {
    constexpr int few = GROUP / 8;  // rows of X whose columns fill a product
    constexpr int swap = GROUP < 128;
    if (T == 1) return nb <= 1024 ? w4_form_of<GROUP, 0, 1, 1, 1, 2>(4) : w4_form_of<GROUP, 0, 1, 1, 2, 2>(4);
    if (T <= few) return nb <= 512 ? w4_form_of<GROUP, 0, 1, few, 1, 2>(4) : nb <= 1024 ? w4_form_of<GROUP, 0, 1, few, 2, 2>(4) : w4_form_of<GROUP, 0, 1, few, 4, 2>(4);
    if constexpr (swap)
        if (T <= 16) return nb <= 512 ? w4_form_of<GROUP, 1, 1, 16, 1, 1>(8) : nb <= 1024 ? w4_form_of<GROUP, 1, 1, 16, 2, 1>(4) : w4_form_of<GROUP, 1, 1, 16, 4, 1>(4);
    if (T > 32 && T <= 48) return nb < 512 ? w4_form_of<GROUP, swap, 3, 48, 1, 1>(8) : w4_form_of<GROUP, swap, 3, 48, 2, 1>(4);
    const long long blocks = (long long)nb * ((T + 31) / 32);
    return blocks < 512 ? w4_form_of<GROUP, swap, 2, 32, 1, 1>(8) : blocks < 1024 ? w4_form_of<GROUP, swap, 2, 32, 2, 1>(4) : w4_form_of<GROUP, swap, 2, 32, 4, 1>(4);
}

int w4_check(const char *fn, const void *codes, const void *scales, const void *dense, int in, int out, int group) {
    ET_REQUIRE(codes && scales && dense, ET_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    ET_REQUIRE(group == 32 || group == 64 || group == 128, ET_ERR_INVALID_ARG, "%s: group=%d must be 32, 64 or 128", fn, group);
    ET_REQUIRE(in > 0 && out > 0, ET_ERR_INVALID_ARG, "%s: in=%d out=%d", fn, in, out);
    ET_REQUIRE(in % group == 0 && out % 16 == 0, ET_ERR_UNSUPPORTED, "%s: in=%d must be a multiple of the group (%d), out=%d of 16", fn, in, group, out);
    ET_REQUIRE((long long)in * out <= 8LL * 0x7fffffff, ET_ERR_UNSUPPORTED, "%s: in=%d out=%d", fn, in, out);
    ET_REQUIRE(((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(dense)) & 15) == 0, ET_ERR_UNSUPPORTED,
               "%s: codes, scales and the matrix must be 16-byte aligned", fn);
    return ET_OK;
}

}  // namespace

}  // namespace et

using namespace et;

extern "C" {

int et_dense_to_w4_f16(const et_f16 *W, uint8_t *codes, et_f16 *scales, int in, int out, int group, et_stream stream) {
    const int st = w4_check("et_dense_to_w4_f16", codes, scales, W, in, out, group);
    if (st != ET_OK) return st;
    const unsigned total = (unsigned)((long long)in * out / 8);
    auto *kernel = group == 32 ? dense_to_w4_kernel<32> : group == 64 ? dense_to_w4_kernel<64> : dense_to_w4_kernel<128>;
    return launch_kernel("dense_to_w4_kernel", kernel, dim3((total + 255) / 256), 256, 0, as_stream(stream), reinterpret_cast<const _Float16 *>(W),
                         reinterpret_cast<unsigned *>(codes), reinterpret_cast<unsigned *>(scales), in, out, total);
}

int et_w4_to_dense_f16(const uint8_t *codes, const et_f16 *scales, et_f16 *W, int in, int out, int group, et_stream stream) {
    const int st = w4_check("et_w4_to_dense_f16", codes, scales, W, in, out, group);
    if (st != ET_OK) return st;
    const unsigned total = (unsigned)((long long)in * out / 8);
    return launch_kernel("w4_to_dense_kernel", w4_to_dense_kernel, dim3((total + 255) / 256), 256, 0, as_stream(stream), reinterpret_cast<const unsigned *>(codes),
                         reinterpret_cast<const unsigned *>(scales), reinterpret_cast<_Float16 *>(W), in, out, group, total);
}

int et_linear_w4_f16(const uint8_t *codes, const et_f16 *scales, int group, const et_f16 *bias, const et_f16 *X, et_f16 *Y, float *Y32, int T, int in,
                     int out, int act, et_stream stream) {
    const int st = w4_check("et_linear_w4_f16", codes, scales, X, in, out, group);
    if (st != ET_OK) return st;
    ET_REQUIRE((Y != nullptr) != (Y32 != nullptr), ET_ERR_INVALID_ARG, "et_linear_w4_f16: exactly one of Y and Y32 must be set");
    ET_REQUIRE(T >= 0, ET_ERR_INVALID_ARG, "et_linear_w4_f16: T=%d", T);
    ET_REQUIRE(act == ET_ACT_NONE || act == ET_ACT_RELU || act == ET_ACT_GELU, ET_ERR_INVALID_ARG, "et_linear_w4_f16: act=%d", act);
    ET_REQUIRE(((reinterpret_cast<uintptr_t>(Y) | reinterpret_cast<uintptr_t>(Y32)) & 15) == 0 && (reinterpret_cast<uintptr_t>(bias) & 7) == 0,
               ET_ERR_UNSUPPORTED, "et_linear_w4_f16: the result must be 16-byte and the bias 8-byte aligned");
    ET_REQUIRE(in <= (1 << 23) && T <= 65535 * 32, ET_ERR_UNSUPPORTED, "et_linear_w4_f16: T=%d in=%d", T, in);
    if (T == 0) return ET_OK;
    const int nb = out / 16;
    const W4Form f = group == 32 ? w4_form<32>(T, nb) : group == 64 ? w4_form<64>(T, nb) : w4_form<128>(T, nb);
    if (f.lds > 64 * 1024) {
        int dev = 0;
        ET_HIP(hipGetDevice(&dev));
        const unsigned long long bit = 1ull << (dev & 63);
        if (!(f.large->load(std::memory_order_relaxed) & bit)) {
            ET_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(f.kernel), hipFuncAttributeMaxDynamicSharedMemorySize, f.lds));
            f.large->fetch_or(bit, std::memory_order_relaxed);
        }
    }
    const W4Args a{codes, reinterpret_cast<const unsigned *>(scales), reinterpret_cast<const _Float16 *>(bias), reinterpret_cast<const _Float16 *>(X),
                   reinterpret_cast<_Float16 *>(Y), Y32, T, in, out, act};
    return launch_kernel("w4_linear_kernel", f.kernel, dim3((unsigned)((nb + f.blocks - 1) / f.blocks), (unsigned)((T + f.rows_x - 1) / f.rows_x)), f.kw * 64u, (size_t)f.lds,
                         as_stream(stream), a);
}

}  // extern "C"
