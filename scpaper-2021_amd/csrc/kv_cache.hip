// A paged cache of keys and values in 4 or 8 bits: written as tokens arrive, read back (layout: et_abi.h).
//
// Eight lanes take one group of 32 channels of four tokens whose positions are 4q .. 4q + 3, bits of the lane: 0 and 1 the token, 3 the eights of channels 0 and 2 or 1 and
// 3 (bit 2: the next group).  A group's extremes are then one rotation inside the 16 lanes, and the four tokens' codes of V, which the cache holds side by side, change places
// inside four neighbouring lanes.  Where a call does not hold all four tokens, the units of 16 bits of those it holds are stored one by one: the bytes of the others are not
// touched.  16 x 1000 tokens of 8 heads of 128, 4 bits, 86 MB read and written: written in 21.3 us, next to memory bound by 19 vector instructions a
// value (16 channels a lane share a group's scale; 8 did not, and took a tenth more), read back in 20.1; 8 bits, 4 x 8192 tokens of 16 heads of 64, 210 MB: 54.7, and 37.8, which is memory's.
// Rows from counts[b] on cost what the others do, all but their stores: with 12256 of the 16000 tokens there, 66 MB, 22.5 and 17.1 us.
#include "group_quant.hip.h"

namespace et {

// n / d of 31-bit n as a product: ceil(2^(31 + l) / d), l = ceil(log2 d), is off by less than 2^l / 2^(31 + l) of it.
struct Divisor {
    unsigned d, magic, shift;
    explicit Divisor(unsigned by = 1) : d(by), shift(0) {
        while ((1ull << shift) < by) shift++;
        magic = (unsigned)((((1ull << (31 + shift)) + by - 1) / by) - 1);  // (- 1: of 1 it would not fit)
    }
    __device__ __forceinline__ unsigned of(unsigned n) const { return (unsigned)(((unsigned long long)n * magic + n) >> (31 + shift)); }
};

struct KvArgs {
    char *k_codes, *v_codes;
    unsigned *k_scales, *v_scales;  // scale in the low half, low in the high one
    const int32_t *table, *starts, *counts;
    const _Float16 *K, *V;
    _Float16 *Kout, *Vout;
    int ldk, ldv;
    int nkv, hd, page, npages, max_pages;
    int n;
    unsigned total;            // units of work of a sequence: groups of a token times groups of four positions that n rows can touch
    Divisor nkvg, groups, page_quads;  // groups of a token, of a head; groups of four positions of a page
};

// Where a unit's tokens lie.
struct KvUnit {
    int group, head;     // of the head's groups; of the heads
    size_t row;          // of this lane's token in the call's matrices, or the nearest that is one
    int count;           // rows of the sequence
    bool mine, all;      // this lane's token is one of the call's and has a place; all four are
    size_t token, quad;  // this lane's token and the first of the four, counted [pages][nkv][page]
    size_t scale;        // the scale of (group, first token of the four)
    int tq, sub;
};

__device__ __forceinline__ KvUnit kv_unit(const KvArgs &a, unsigned unit) {
    KvUnit u;
    const int b = blockIdx.y;
    u.tq = threadIdx.x & 3;
    u.sub = threadIdx.x >> 3 & 1;
    const bool none = unit >= a.total;  // (of the pair of units that 16 lanes take, the second may be none: its lanes stay for the rotations, on the last unit)
    if (none) unit = a.total - 1;
    const unsigned q = a.nkvg.of(unit), g = unit - q * a.nkvg.d;
    u.head = (int)a.groups.of(g);
    u.group = (int)(g - u.head * a.groups.d);
    const int start = a.starts ? a.starts[b] : 0, count = a.counts ? min(max(a.counts[b], 0), a.n) : a.n;
    // floor(start / 4) + q also below zero; as 64-bit numbers where start + count pass 2^31
    const long long quad = (start >> 2) + (long long)q;
    const long long i0 = quad * 4 - start;  // row of the first of the four
    const long long i = i0 + u.tq;
    const bool reach = quad >= 0 && quad < (1ll << 29);
    const unsigned page_at = a.page_quads.of(reach ? (unsigned)quad : 0u), off = ((reach ? (unsigned)quad : 0u) - page_at * a.page_quads.d) * 4;
    int page = -1;
    if (reach && page_at < (unsigned)a.max_pages) page = a.table[(size_t)b * a.max_pages + page_at];
    const bool placed = page >= 0 && page < a.npages;
    u.mine = !none && placed && i >= 0 && i < count;
    u.all = !none && placed && i0 >= 0 && i0 + 3 < count;
    const size_t ph = (size_t)(placed ? page : 0) * a.nkv + u.head;
    u.quad = ph * a.page + (placed ? off : 0u);
    u.token = u.quad + u.tq;
    u.scale = (ph * a.groups.d + u.group) * a.page + (placed ? off : 0u);
    u.row = (size_t)b * a.n + (size_t)min(max(i, 0LL), (long long)max(count - 1, 0));
    u.count = count;
    return u;
}

template <int CTRL> __device__ __forceinline__ unsigned dpp_bits(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}

template <int BITS> __device__ __forceinline__ void kv_quantise(const h8 (&x)[2], unsigned (&codes)[BITS / 2], unsigned &scale_low) {
    unsigned magnitude, more, tiny, tiny_more;
    h2 e = extremes(x[0], magnitude, tiny);
    const h2 f = extremes(x[1], more, tiny_more);
    extremes_of(e, magnitude, f, more);
    extremes_across<kDppRowRor8>(e, magnitude);
    quantise<BITS, 2>(codes, scale_low, x, e, magnitude, least_of(tiny, tiny_more));
}

// Between pairs of lanes: the first of a pair ends with `first` of both, the second with `second` of both, in the lanes' order.
template <int CTRL> __device__ __forceinline__ void trade(unsigned &mine, unsigned &other, unsigned first, unsigned second, bool is_second) {
    const unsigned got = dpp_bits<CTRL>(is_second ? first : second);
    mine = is_second ? got : first;
    other = is_second ? second : got;
}

template <int BITS> __global__ __launch_bounds__(256) void kv_write_kernel(const KvArgs a) {
    const unsigned unit = blockIdx.x * 32 + (threadIdx.x >> 4) * 2 + (threadIdx.x >> 2 & 1);
    const KvUnit u = kv_unit(a, unit);
    const int col = u.head * a.hd + u.group * ET_KV_GROUP + u.sub * 8;
    if (u.count <= 0) return;  // (of the whole workgroup's sequence)
    // (lanes whose token is none of the call's take the nearest row that is)
    const _Float16 *from_k = a.K + u.row * a.ldk + col, *from_v = a.V + u.row * a.ldv + col;
    const h8 k[2] = {*reinterpret_cast<const h8 *>(from_k), *reinterpret_cast<const h8 *>(from_k + 16)};
    const h8 v[2] = {*reinterpret_cast<const h8 *>(from_v), *reinterpret_cast<const h8 *>(from_v + 16)};
    constexpr int W = BITS / 4;  // words of eight codes
    unsigned c[2 * W], sl;
    const int token_bytes = a.hd * BITS / 8, at = (u.group * ET_KV_GROUP + u.sub * 8) * BITS / 8;
    kv_quantise<BITS>(k, c, sl);
    if (u.mine) {
        char *to = a.k_codes + u.token * token_bytes + at;
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int w = 0; w < W; w++) *reinterpret_cast<unsigned *>(to + e * 2 * BITS + w * 4) = c[e * W + w];
        if (u.sub == 0) a.k_scales[u.scale + u.tq] = sl;
    }
    kv_quantise<BITS>(v, c, sl);
    // The four tokens' units from at / 2 on, [unit][token]: words of two units change places between the four lanes, which each store 16 bytes (8 with 4 bits) in one
    // piece.  Word by word, 4 bytes a lane, the stores were four times as many requests: 8 bits, 4 x 8192 tokens of 16 heads of 64 60.6 us instead of 54.6.
    char *to = a.v_codes + u.quad * token_bytes + (size_t)at * 4;
    const bool odd = u.tq & 1, high = u.tq & 2;
    unsigned x[2 * W];
#pragma unroll
    for (int i = 0; i < 2 * W; i += 2) trade<kDppQuadXor1>(x[i], x[i + 1], c[i], c[i + 1], odd);  // -> word i, of odd lanes i + 1, of this lane and its neighbour, by token
    constexpr unsigned lows = 0x05040100u, highs = 0x07060302u;
    if constexpr (BITS == 8) {
        unsigned y[4];
        trade<kDppQuadXor2>(y[0], y[2], x[0], x[2], high);
        trade<kDppQuadXor2>(y[1], y[3], x[1], x[3], high);
        if (u.all)
            *reinterpret_cast<uint4 *>(to + (u.tq >> 1) * 64 + odd * 16) = uint4{__builtin_amdgcn_perm(y[1], y[0], lows), __builtin_amdgcn_perm(y[3], y[2], lows),
                                                                                 __builtin_amdgcn_perm(y[1], y[0], highs), __builtin_amdgcn_perm(y[3], y[2], highs)};
    } else {
        unsigned y[2];
        trade<kDppQuadXor2>(y[0], y[1], __builtin_amdgcn_perm(x[1], x[0], lows), __builtin_amdgcn_perm(x[1], x[0], highs), high);
        if (u.all) *reinterpret_cast<uint2 *>(to + odd * 32 + (u.tq >> 1) * 8) = uint2{y[0], y[1]};
    }
    if (!u.all && u.mine) {
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int w = 0; w < W; w++) {
                char *here = to + e * 8 * BITS + w * 16 + u.tq * 2;
                *reinterpret_cast<unsigned short *>(here) = (unsigned short)c[e * W + w];
                *reinterpret_cast<unsigned short *>(here + 8) = (unsigned short)(c[e * W + w] >> 16);
            }
    }
    if (u.mine && u.sub == 0) a.v_scales[u.scale + u.tq] = sl;
}

template <int BITS> __device__ __forceinline__ h8 kv_values(const unsigned *c, unsigned scale_low) {
    const float s = f16_bits_value(scale_low & 0xffffu), lo = f16_bits_value(scale_low >> 16);
    h8 x;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = step_value((float)((c[i * BITS / 32] >> (i * BITS % 32)) & (BITS == 4 ? 15u : 255u)), lo, s);
    return x;
}

template <int BITS> __global__ __launch_bounds__(256) void kv_read_kernel(const KvArgs a) {
    const unsigned unit = blockIdx.x * 32 + (threadIdx.x >> 4) * 2 + (threadIdx.x >> 2 & 1);
    const KvUnit u = kv_unit(a, unit);
    const int col = u.head * a.hd + u.group * ET_KV_GROUP + u.sub * 8;
    constexpr int W = BITS / 4;
    unsigned c[2 * W] = {}, d[2 * W] = {};
    unsigned k_sl = 0, v_sl = 0;
    const int token_bytes = a.hd * BITS / 8, at = (u.group * ET_KV_GROUP + u.sub * 8) * BITS / 8;
    if (a.Kout && u.mine) {
        const char *from = a.k_codes + u.token * token_bytes + at;
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int w = 0; w < W; w++) c[e * W + w] = *reinterpret_cast<const unsigned *>(from + e * 2 * BITS + w * 4);
        k_sl = a.k_scales[u.scale + u.tq];
    }
    if (a.Vout) {
        // (the page of a token of this call holds all four: lanes whose token is not the call's read too, for their neighbours, or read page 0 and store nothing)
        const char *from = a.v_codes + u.quad * token_bytes + (size_t)at * 4;
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int w = 0; w < W; w++) d[e * W + w] = *reinterpret_cast<const unsigned *>(from + e * 8 * BITS + w * 16 + u.tq * 4);
        v_sl = a.v_scales[u.scale + u.tq];
    }
    if (a.Kout && u.mine) {
        _Float16 *to = a.Kout + u.row * a.ldk + col;
        *reinterpret_cast<h8 *>(to) = kv_values<BITS>(c, k_sl);
        *reinterpret_cast<h8 *>(to + 16) = kv_values<BITS>(c + W, k_sl);
    }
    if (!a.Vout) return;
#pragma unroll
    for (int w = 0; w < 2 * W; w++) {
        const unsigned first = dpp_bits<0x50>(d[w]), second = dpp_bits<0xFA>(d[w]);  // quad_perm [0,0,1,1] and [2,2,3,3]
        c[w] = u.tq & 1 ? (first >> 16) | (second & 0xffff0000u) : (first & 0xffffu) | second << 16;
    }
    if (u.mine) {
        _Float16 *to = a.Vout + u.row * a.ldv + col;
        *reinterpret_cast<h8 *>(to) = kv_values<BITS>(c, v_sl);
        *reinterpret_cast<h8 *>(to + 16) = kv_values<BITS>(c + W, v_sl);
    }
}

int kv_check_cache(const char *fn, const et_kv_cache *c, const int32_t *table, int max_pages, int B, int n) {
    ET_REQUIRE(c && c->k_codes && c->k_scales && c->v_codes && c->v_scales && table, ET_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    ET_REQUIRE(c->nkv > 0 && c->hd > 0 && c->page > 0 && c->npages > 0 && max_pages > 0 && B >= 0 && n >= 0, ET_ERR_INVALID_ARG,
               "%s: nkv=%d hd=%d page=%d npages=%d max_pages=%d B=%d n=%d", fn, c->nkv, c->hd, c->page, c->npages, max_pages, B, n);
    ET_REQUIRE(c->bits == 4 || c->bits == 8, ET_ERR_INVALID_ARG, "%s: bits=%d must be 4 or 8", fn, c->bits);
    ET_REQUIRE(c->hd % ET_KV_GROUP == 0 && c->hd <= 256, ET_ERR_UNSUPPORTED, "%s: hd=%d must be a multiple of %d, at most 256", fn, c->hd, ET_KV_GROUP);
    ET_REQUIRE(c->page % 16 == 0, ET_ERR_UNSUPPORTED, "%s: page=%d must be a multiple of 16", fn, c->page);
    ET_REQUIRE(((reinterpret_cast<uintptr_t>(c->k_codes) | reinterpret_cast<uintptr_t>(c->k_scales) | reinterpret_cast<uintptr_t>(c->v_codes) |
                 reinterpret_cast<uintptr_t>(c->v_scales)) & 15) == 0, ET_ERR_UNSUPPORTED, "%s: the cache's buffers must be 16-byte aligned", fn);
    ET_REQUIRE((reinterpret_cast<uintptr_t>(table) & 3) == 0, ET_ERR_UNSUPPORTED, "%s: table must be 4-byte aligned", fn);
    // (a tile of keys may reach 64 positions beyond: positions stay 32-bit numbers)
    ET_REQUIRE((long long)max_pages * c->page <= 0x7fffff80LL, ET_ERR_UNSUPPORTED, "%s: max_pages * page = %lld positions", fn, (long long)max_pages * c->page);
    ET_REQUIRE((long long)c->nkv * c->hd <= (1 << 24) && (long long)c->nkv * c->hd * c->page / 8 * c->bits < (1LL << 31), ET_ERR_UNSUPPORTED,
               "%s: nkv * hd = %lld, %d tokens a page", fn, (long long)c->nkv * c->hd, c->page);
    return ET_OK;
}

namespace {

int kv_args(const char *fn, KvArgs &a, const et_kv_cache *cache, const int32_t *table, int max_pages, const int32_t *starts, const int32_t *counts,
            const void *K, const void *V, int ldk, int ldv, int B, int n) {
    const int st = kv_check_cache(fn, cache, table, max_pages, B, n);
    if (st != ET_OK) return st;
    const int width = cache->nkv * cache->hd;
    ET_REQUIRE((!K || ldk >= width) && (!V || ldv >= width), ET_ERR_INVALID_ARG, "%s: row strides %d, %d below nkv * hd = %d", fn, ldk, ldv, width);
    ET_REQUIRE((!K || ldk % 8 == 0) && (!V || ldv % 8 == 0), ET_ERR_UNSUPPORTED, "%s: row strides must be multiples of 8", fn);
    ET_REQUIRE(((reinterpret_cast<uintptr_t>(K) | reinterpret_cast<uintptr_t>(V)) & 15) == 0, ET_ERR_UNSUPPORTED, "%s: K and V must be 16-byte aligned", fn);
    a.k_codes = static_cast<char *>(cache->k_codes);
    a.v_codes = static_cast<char *>(cache->v_codes);
    a.k_scales = reinterpret_cast<unsigned *>(cache->k_scales);
    a.v_scales = reinterpret_cast<unsigned *>(cache->v_scales);
    a.table = table;
    a.starts = starts;
    a.counts = counts;
    a.K = a.V = nullptr;
    a.Kout = a.Vout = nullptr;
    a.ldk = ldk;
    a.ldv = ldv;
    a.nkv = cache->nkv;
    a.hd = cache->hd;
    a.page = cache->page;
    a.npages = cache->npages;
    a.max_pages = max_pages;
    a.n = n;
    a.nkvg = Divisor((unsigned)(width / ET_KV_GROUP));
    a.groups = Divisor((unsigned)(cache->hd / ET_KV_GROUP));
    a.page_quads = Divisor((unsigned)(cache->page / 4));
    // n positions from any start touch at most this many groups of four; eight threads a unit, and a launch counts its threads in 32 bits
    const long long quads = starts ? (n + 2LL) / 4 + 1 : (n + 3LL) / 4, total = n == 0 ? 0 : quads * a.nkvg.d;
    ET_REQUIRE(B <= 65535 && total <= (1LL << 29) - 32, ET_ERR_UNSUPPORTED, "%s: B=%d n=%d", fn, B, n);
    a.total = (unsigned)total;
    return ET_OK;
}

}  // namespace

}  // namespace et

using namespace et;

extern "C" {

int et_kv_write_f16(const et_kv_cache *cache, const int32_t *table, int max_pages, const int32_t *starts, const int32_t *counts, const et_f16 *K,
                    const et_f16 *V, int ldk, int ldv, int B, int n, et_stream stream) {
    ET_REQUIRE(K && V, ET_ERR_INVALID_ARG, "et_kv_write_f16: NULL pointer");
    KvArgs a;
    const int st = kv_args("et_kv_write_f16", a, cache, table, max_pages, starts, counts, K, V, ldk, ldv, B, n);
    if (st != ET_OK || a.total == 0 || B == 0) return st;
    a.K = reinterpret_cast<const _Float16 *>(K);
    a.V = reinterpret_cast<const _Float16 *>(V);
    return launch_kernel("kv_write_kernel", cache->bits == 4 ? kv_write_kernel<4> : kv_write_kernel<8>, dim3((a.total + 31) / 32, (unsigned)B), 256, 0, as_stream(stream), a);
}

int et_kv_read_f16(const et_kv_cache *cache, const int32_t *table, int max_pages, const int32_t *starts, const int32_t *counts, et_f16 *K, et_f16 *V,
                   int ldk, int ldv, int B, int n, et_stream stream) {
    KvArgs a;
    const int st = kv_args("et_kv_read_f16", a, cache, table, max_pages, starts, counts, K, V, ldk, ldv, B, n);
    if (st != ET_OK || a.total == 0 || B == 0 || (!K && !V)) return st;
    a.Kout = reinterpret_cast<_Float16 *>(K);
    a.Vout = reinterpret_cast<_Float16 *>(V);
    return launch_kernel("kv_read_kernel", cache->bits == 4 ? kv_read_kernel<4> : kv_read_kernel<8>, dim3((a.total + 31) / 32, (unsigned)B), 256, 0, as_stream(stream), a);
}

}  // extern "C"
