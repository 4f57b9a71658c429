// Linear with 4-bit weights, a scale and a lowest value for every 32, 64 or 128 input features of an output feature (layout: et_abi.h).
#include "group_quant.hip.h"

namespace et {

// Sixteen lanes a group of an output feature: group / 16 values each, as words of codes where there are eight of them.
template <int GROUP> __global__ __launch_bounds__(256) void dense_to_w4_kernel(const _Float16 *W, unsigned *codes, unsigned *scales, int in, int out, unsigned total) {
    // a lane holds eight values; GROUP / 8 neighbouring lanes (4, 8 or 16) a group
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    if (i >= total) return;  // (total is a multiple of GROUP / 8, and so are a wave's first and last)
    const h8 x = reinterpret_cast<const h8 *>(W)[i];
    float lo = (float)x[0], hi = lo, bad = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const float v = (float)x[k];
        lo = fminf(lo, v);
        hi = fmaxf(hi, v);
        bad = __builtin_fmaf(v, 0.0f, bad);
    }
    auto across = [&](auto move) {
        lo = fminf(lo, move(lo));
        hi = fmaxf(hi, move(hi));
        bad += move(bad);
    };
    across(dpp_move<kDppQuadXor1>);
    across(dpp_move<kDppQuadXor2>);
    if constexpr (GROUP >= 64) across(dpp_move<0x141>);   // row_half_mirror: the other four of eight
    if constexpr (GROUP >= 128) across(dpp_move<0x128>);  // row_ror:8
    const bool finite = bad == 0.0f;
    lo = finite ? lo : 0.0f;
    hi = finite ? hi : 0.0f;
    const unsigned sb = group_scale_bits(lo, hi, 15.0f);
    const float s = f16_bits_value(sb), inv = s > 0.0f ? 1.0f / s : 0.0f;
    unsigned word = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) word |= (finite ? (unsigned)(int)nearest_step((float)x[k], lo, s, inv) : 0u) << (4 * k);
    codes[i] = word;
    const unsigned per_row = (unsigned)in / 8, o = i / per_row, at = i - o * per_row;
    const unsigned low_bits = finite ? __builtin_bit_cast(unsigned short, (_Float16)lo) : (unsigned short)0x7E00;
    if (at % (GROUP / 8) == 0) scales[(size_t)(at / (GROUP / 8)) * out + o] = sb | low_bits << 16;
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
    const unsigned *scales;
    const _Float16 *bias, *X;
    _Float16 *Y;
    float *Y32;
    int T, in, out, group, act;
};

// One wave an output value.
__global__ __launch_bounds__(256) void w4_linear_plain_kernel(const W4Args a) {
    const int lane = threadIdx.x & 63, o = blockIdx.x * 4 + (threadIdx.x >> 6);
    const size_t t = blockIdx.y;
    const _Float16 *x = a.X + t * a.in;
    float y = 0.0f;
    for (int i = lane; i < a.in; i += 64) {
        const unsigned sl = a.scales[(size_t)(i / a.group) * a.out + o];
        const unsigned c = (a.codes[((size_t)o * a.in + i) / 2] >> (i % 2 * 4)) & 15u;
        y += (float)x[i] * __builtin_fmaf(f16_bits_value(sl & 0xffffu), (float)c, f16_bits_value(sl >> 16));
    }
    y = apply_act(wave_sum(y) + (a.bias ? (float)a.bias[o] : 0.0f), a.act);
    if (lane != 0) return;
    if (a.Y) a.Y[t * a.out + o] = (_Float16)y;
    else a.Y32[t * a.out + o] = y;
}

namespace {

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
    ET_REQUIRE(T <= 65535, ET_ERR_UNSUPPORTED, "et_linear_w4_f16: T=%d", T);
    if (T == 0) return ET_OK;
    W4Args a{codes, reinterpret_cast<const unsigned *>(scales), reinterpret_cast<const _Float16 *>(bias), reinterpret_cast<const _Float16 *>(X),
             reinterpret_cast<_Float16 *>(Y), Y32, T, in, out, group, act};
    return launch_kernel("w4_linear_plain_kernel", w4_linear_plain_kernel, dim3(out / 4, T), 256, 0, as_stream(stream), a);
}

}  // extern "C"
