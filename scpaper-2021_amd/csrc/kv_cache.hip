// A paged cache of keys and values in 4 or 8 bits: written as tokens arrive, read back (layout: et_abi.h).
//
// Sixteen lanes take one group of 32 channels of four tokens whose positions are 4q .. 4q + 3: lane % 4 the token, lane / 4 eight of the
// channels.  A group's extremes are then two rotations inside the 16 lanes, and the four tokens' codes of V, which the cache holds side by
// side, change places inside four neighbouring lanes.  Where a call does not hold all four tokens, the units of 16 bits of those it
// holds are stored one by one: the bytes of the others are not touched.
#include "group_quant.hip.h"

namespace et {

struct KvArgs {
    char *k_codes, *v_codes;
    unsigned *k_scales, *v_scales;  // scale in the low half, low in the high one
    const int32_t *table, *starts, *counts;
    const _Float16 *K, *V;
    _Float16 *Kout, *Vout;
    int ldk, ldv;
    int nkv, hd, page, npages, max_pages;
    int n, quads;         // rows of a sequence; groups of four positions that they can touch
    unsigned nkvg, total; // groups of a token; units of work
};

template <int CTRL> __device__ __forceinline__ unsigned dpp_bits(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}

// Where a unit's tokens lie.
struct KvUnit {
    int group, head;   // of the head's groups; of the heads
    long long row;     // row of this lane's token in the call's matrices
    bool mine, all;    // this lane's token is one of the call's and has a place; all four are
    size_t token, quad;  // token's index [pages][nkv][page] with page/head resolved, and that of the first of the four
    size_t scale;      // index of the scale of (group, first token of the four)
    int tq, sub;
};

__device__ __forceinline__ KvUnit kv_unit(const KvArgs &a, unsigned unit) {
    KvUnit u;
    const int lane = threadIdx.x & 15;
    u.tq = lane & 3;
    u.sub = lane >> 2;
    const unsigned g = unit % a.nkvg, rest = unit / a.nkvg;
    const int quad = (int)(rest % (unsigned)a.quads), b = (int)(rest / (unsigned)a.quads);
    const int groups = a.hd / ET_KV_GROUP;
    u.head = (int)g / groups;
    u.group = (int)g - u.head * groups;
    const long long start = a.starts ? a.starts[b] : 0;
    const int count = a.counts ? min(max(a.counts[b], 0), a.n) : a.n;
    // floor(start / 4) also below zero
    const long long pos0 = ((start >> 2) + quad) * 4;
    const long long i = pos0 + u.tq - start;
    const long long pidx = pos0 / a.page;
    int page = -1;
    if (pos0 >= 0 && pidx < a.max_pages) page = a.table[(size_t)b * a.max_pages + (size_t)pidx];
    const bool placed = page >= 0 && page < a.npages;
    const bool inside = i >= 0 && i < count;
    u.mine = placed && inside;
    const long long i0 = pos0 - start;
    u.all = placed && i0 >= 0 && i0 + 3 < count;
    const int off = placed ? (int)(pos0 - pidx * a.page) : 0;
    const size_t ph = (size_t)(placed ? page : 0) * a.nkv + u.head;
    u.quad = ph * a.page + off;
    u.token = u.quad + u.tq;
    u.scale = (ph * groups + u.group) * a.page + off;
    u.row = (long long)b * a.n + i;
    return u;
}

__device__ __forceinline__ float row16_min(float v) {
    v = fminf(v, dpp_move<kRowRor4>(v));
    return fminf(v, dpp_move<kRowRor8>(v));
}
__device__ __forceinline__ float row16_max(float v) {
    v = fmaxf(v, dpp_move<kRowRor4>(v));
    return fmaxf(v, dpp_move<kRowRor8>(v));
}

// Codes of eight values, and the group's (scale, low).
template <int BITS> __device__ __forceinline__ void kv_quantise(const h8 x, unsigned (&codes)[BITS / 4], unsigned &scale_low) {
    float lo = (float)x[0], hi = lo, bad = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float v = (float)x[i];
        lo = fminf(lo, v);
        hi = fmaxf(hi, v);
        bad = __builtin_fmaf(v, 0.0f, bad);  // NaN from the first NaN or infinity on
    }
    lo = row16_min(lo);
    hi = row16_max(hi);
    bad += dpp_move<kRowRor4>(bad);
    bad += dpp_move<kRowRor8>(bad);
    const bool finite = bad == 0.0f;
    lo = finite ? lo : 0.0f;
    hi = finite ? hi : 0.0f;
    const unsigned sb = group_scale_bits(lo, hi, BITS == 4 ? 15.0f : 255.0f);
    const float s = f16_bits_value(sb), inv = s > 0.0f ? 1.0f / s : 0.0f;
#pragma unroll
    for (int w = 0; w < BITS / 4; w++) codes[w] = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const unsigned c = finite ? (unsigned)(int)nearest_step((float)x[i], lo, s, inv) : 0u;
        codes[i * BITS / 32] |= c << (i * BITS % 32);
    }
    const unsigned short low_bits = finite ? __builtin_bit_cast(unsigned short, (_Float16)lo) : (unsigned short)0x7E00;
    scale_low = sb | (unsigned)low_bits << 16;
}

template <int BITS> __global__ __launch_bounds__(256) void kv_write_kernel(const KvArgs a) {
    const unsigned unit = blockIdx.x * 16 + (threadIdx.x >> 4);
    if (unit >= a.total) return;
    const KvUnit u = kv_unit(a, unit);
    const int col = u.head * a.hd + u.group * ET_KV_GROUP + u.sub * 8;
    h8 k = {0, 0, 0, 0, 0, 0, 0, 0}, v = k;
    if (u.mine) {
        k = *reinterpret_cast<const h8 *>(a.K + (size_t)u.row * a.ldk + col);
        v = *reinterpret_cast<const h8 *>(a.V + (size_t)u.row * a.ldv + col);
    }
    constexpr int W = BITS / 4;  // words of a lane's eight codes
    unsigned c[W], sl;
    const int token_bytes = a.hd * BITS / 8, at = (u.group * ET_KV_GROUP + u.sub * 8) * BITS / 8;
    kv_quantise<BITS>(k, c, sl);
    if (u.mine) {
        unsigned *to = reinterpret_cast<unsigned *>(a.k_codes + u.token * token_bytes + at);
#pragma unroll
        for (int w = 0; w < W; w++) to[w] = c[w];
        if (u.sub == 0) a.k_scales[u.scale + u.tq] = sl;
    }
    kv_quantise<BITS>(v, c, sl);
    // the four tokens' units from at / 2 on, [unit][token]
    char *to = a.v_codes + u.quad * token_bytes + (size_t)at * 4;
    if (u.all) {
#pragma unroll
        for (int w = 0; w < W; w++) {
            // lane m of four stores unit m / 2 of tokens 2 (m % 2) and the next
            const unsigned first = dpp_bits<0x88>(c[w]), second = dpp_bits<0xDD>(c[w]);  // quad_perm [0,2,0,2] and [1,3,1,3]
            const unsigned word = u.tq & 2 ? (first >> 16) | (second & 0xffff0000u) : (first & 0xffffu) | second << 16;
            *reinterpret_cast<unsigned *>(to + w * 16 + u.tq * 4) = word;
        }
    } else if (u.mine) {
#pragma unroll
        for (int w = 0; w < W; w++) {
            *reinterpret_cast<unsigned short *>(to + w * 16 + u.tq * 2) = (unsigned short)c[w];
            *reinterpret_cast<unsigned short *>(to + w * 16 + 8 + u.tq * 2) = (unsigned short)(c[w] >> 16);
        }
    }
    if (u.mine && u.sub == 0) a.v_scales[u.scale + u.tq] = sl;
}

template <int BITS> __device__ __forceinline__ h8 kv_values(const unsigned (&c)[BITS / 4], unsigned scale_low) {
    const float s = f16_bits_value(scale_low & 0xffffu), lo = f16_bits_value(scale_low >> 16);
    h8 x;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = step_value((float)((c[i * BITS / 32] >> (i * BITS % 32)) & (BITS == 4 ? 15u : 255u)), lo, s);
    return x;
}

template <int BITS> __global__ __launch_bounds__(256) void kv_read_kernel(const KvArgs a) {
    const unsigned unit = blockIdx.x * 16 + (threadIdx.x >> 4);
    if (unit >= a.total) return;
    const KvUnit u = kv_unit(a, unit);
    const int col = u.head * a.hd + u.group * ET_KV_GROUP + u.sub * 8;
    constexpr int W = BITS / 4;
    unsigned c[W] = {}, d[W] = {};
    const int token_bytes = a.hd * BITS / 8, at = (u.group * ET_KV_GROUP + u.sub * 8) * BITS / 8;
    if (a.Kout && u.mine) {
        const unsigned *from = reinterpret_cast<const unsigned *>(a.k_codes + u.token * token_bytes + at);
#pragma unroll
        for (int w = 0; w < W; w++) c[w] = from[w];
        *reinterpret_cast<h8 *>(a.Kout + (size_t)u.row * a.ldk + col) = kv_values<BITS>(c, a.k_scales[u.scale + u.tq]);
    }
    if (!a.Vout) return;
    // (the page of a token of this call holds all four: lanes whose token is not the call's read too, for their neighbours, or read page 0 and store nothing)
    const char *from = a.v_codes + u.quad * token_bytes + (size_t)at * 4;
#pragma unroll
    for (int w = 0; w < W; w++) d[w] = *reinterpret_cast<const unsigned *>(from + w * 16 + u.tq * 4);
    const unsigned sl = a.v_scales[u.scale + u.tq];
#pragma unroll
    for (int w = 0; w < W; w++) {
        const unsigned first = dpp_bits<0x50>(d[w]), second = dpp_bits<0xFA>(d[w]);  // quad_perm [0,0,1,1] and [2,2,3,3]
        c[w] = u.tq & 1 ? (first >> 16) | (second & 0xffff0000u) : (first & 0xffffu) | second << 16;
    }
    if (u.mine) *reinterpret_cast<h8 *>(a.Vout + (size_t)u.row * a.ldv + col) = kv_values<BITS>(c, sl);
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
    ET_REQUIRE((long long)max_pages * c->page <= 0x7fffffffLL, ET_ERR_UNSUPPORTED, "%s: max_pages * page = %lld positions", fn, (long long)max_pages * c->page);
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
    // n positions from any start touch at most this many groups of four
    a.quads = starts ? (int)((n + 2LL) / 4) + 1 : (int)((n + 3LL) / 4);
    a.nkvg = (unsigned)(width / ET_KV_GROUP);
    const long long total = (long long)B * a.quads * a.nkvg;
    ET_REQUIRE(total <= 0x7fffffffLL, ET_ERR_UNSUPPORTED, "%s: %lld groups in one call", fn, total * 4);
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
    if (st != ET_OK || a.total == 0 || n == 0) return st;
    a.K = reinterpret_cast<const _Float16 *>(K);
    a.V = reinterpret_cast<const _Float16 *>(V);
    return launch_kernel("kv_write_kernel", cache->bits == 4 ? kv_write_kernel<4> : kv_write_kernel<8>, dim3((a.total + 15) / 16), 256, 0, as_stream(stream), a);
}

int et_kv_read_f16(const et_kv_cache *cache, const int32_t *table, int max_pages, const int32_t *starts, const int32_t *counts, et_f16 *K, et_f16 *V,
                   int ldk, int ldv, int B, int n, et_stream stream) {
    KvArgs a;
    const int st = kv_args("et_kv_read_f16", a, cache, table, max_pages, starts, counts, K, V, ldk, ldv, B, n);
    if (st != ET_OK || a.total == 0 || n == 0 || (!K && !V)) return st;
    a.Kout = reinterpret_cast<_Float16 *>(K);
    a.Vout = reinterpret_cast<_Float16 *>(V);
    return launch_kernel("kv_read_kernel", cache->bits == 4 ? kv_read_kernel<4> : kv_read_kernel<8>, dim3((a.total + 15) / 16), 256, 0, as_stream(stream), a);
}

}  // extern "C"
