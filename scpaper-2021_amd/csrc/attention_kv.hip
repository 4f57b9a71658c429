// Attention over a cache of keys and values in 4 or 8 bits (layout: et_abi.h).
#include <math.h>

#include "group_quant.hip.h"

namespace et {

int kv_check_cache(const char *fn, const et_kv_cache *c, const int32_t *table, int max_pages, int B, int n);

struct KvMhaArgs {
    const unsigned char *k_codes;
    const unsigned short *v_codes;
    const unsigned *k_scales, *v_scales;
    const int32_t *table, *starts, *counts;
    const _Float16 *Q;
    _Float16 *Z;
    int ldq, ldz;
    int nkv, hd, page, npages, max_pages;
    int n, nh, causal;
    float scale_log2e;
};

// One wave a (row, head): 64 keys at a time, one a lane; then the channels of Z one a lane.
template <int BITS> __global__ __launch_bounds__(64) void mha_kv_plain_kernel(const KvMhaArgs a) {
    const int lane = threadIdx.x;
    const int h = blockIdx.x, row = blockIdx.y, b = blockIdx.z;
    const long long start = a.starts ? a.starts[b] : 0;
    const int count = a.counts ? min(max(a.counts[b], 0), a.n) : a.n;
    if (row >= count) return;
    const int kv = h / (a.nh / a.nkv), groups = a.hd / ET_KV_GROUP;
    long long end = a.causal ? start + row + 1 : start + count;
    end = min(end, (long long)a.max_pages * a.page);
    const _Float16 *q = a.Q + ((size_t)b * a.n + row) * a.ldq + h * a.hd;
    float m = -INFINITY, l = 0.0f, acc[4] = {0, 0, 0, 0};
    for (long long k0 = 0; k0 < end; k0 += 64) {
        const long long pos = k0 + lane;
        int page = -1;
        if (pos < end) page = a.table[(size_t)b * a.max_pages + (size_t)(pos / a.page)];
        const bool seen = page >= 0 && page < a.npages;
        const int off = (int)(pos % a.page);
        const size_t ph = (size_t)(seen ? page : 0) * a.nkv + kv;
        float score = -INFINITY;
        if (seen) {
            const unsigned char *c = a.k_codes + (ph * a.page + off) * (a.hd * BITS / 8);
            score = 0.0f;
            for (int g = 0; g < groups; g++) {
                const unsigned sl = a.k_scales[(ph * groups + g) * a.page + off];
                float dot = 0.0f, sum = 0.0f;
                for (int d = 0; d < 32; d++) {
                    const int ch = g * 32 + d;
                    const float x = (float)q[ch];
                    dot += x * (float)(BITS == 4 ? (c[ch / 2] >> (ch % 2 * 4)) & 15 : c[ch]);
                    sum += x;
                }
                score += f16_bits_value(sl & 0xffffu) * dot + f16_bits_value(sl >> 16) * sum;
            }
            score *= a.scale_log2e;
        }
        const float top = fmaxf(m, wave_max(score));
        if (top == -INFINITY) continue;
        const float keep = exp2f(m - top), p = exp2f(score - top);
        m = top;
        l = l * keep + wave_sum(p);
        for (int i = 0; i < 4; i++) acc[i] *= keep;
        const int last = (int)min(64LL, end - k0);
        for (int t = 0; t < last; t++) {
            const float pt = lane_value(p, t);
            const int tp = __builtin_amdgcn_readlane(seen ? page : -1, t), to = __builtin_amdgcn_readlane(off, t);
            if (tp < 0) continue;
            const size_t th = (size_t)tp * a.nkv + kv;
            const unsigned short *units = a.v_codes + (th * a.page + (to & ~3)) * (a.hd * BITS / 16) + (to & 3);
            for (int i = 0; i < 4; i++) {
                const int d = lane + 64 * i;
                if (d >= a.hd) break;
                const unsigned sl = a.v_scales[(th * groups + d / 32) * a.page + to];
                const unsigned u = units[(d * BITS / 16) * 4];
                const float c = (float)((u >> (d * BITS % 16)) & (BITS == 4 ? 15u : 255u));
                acc[i] += pt * __builtin_fmaf(f16_bits_value(sl & 0xffffu), c, f16_bits_value(sl >> 16));
            }
        }
    }
    for (int i = 0; i < 4; i++) {
        const int d = lane + 64 * i;
        if (d < a.hd) a.Z[((size_t)b * a.n + row) * a.ldz + h * a.hd + d] = (_Float16)(l > 0.0f ? acc[i] / l : 0.0f);
    }
}

}  // namespace et

using namespace et;

extern "C" {

int et_mha_kv_workspace(const et_kv_cache *cache, int max_pages, int B, int n, int nh, size_t *bytes) {
    ET_REQUIRE(bytes, ET_ERR_INVALID_ARG, "et_mha_kv_workspace: NULL pointer");
    static const int32_t any = 0;
    const int st = kv_check_cache("et_mha_kv_workspace", cache, &any, max_pages, B, n);
    if (st != ET_OK) return st;
    *bytes = 0;
    return ET_OK;
}

int et_mha_kv_f16(const et_kv_cache *cache, const int32_t *table, int max_pages, const int32_t *starts, const int32_t *counts, const et_f16 *Q, int ldq,
                  et_f16 *Z, int ldz, int B, int n, int nh, float scale, int flags, void *workspace, size_t workspace_bytes, et_stream stream) {
    ET_REQUIRE(Q && Z, ET_ERR_INVALID_ARG, "et_mha_kv_f16: NULL pointer");
    const int st = kv_check_cache("et_mha_kv_f16", cache, table, max_pages, B, n);
    if (st != ET_OK) return st;
    ET_REQUIRE((flags & ~ET_MHA_CAUSAL) == 0, ET_ERR_INVALID_ARG, "et_mha_kv_f16: flags=%d", flags);
    ET_REQUIRE(nh > 0 && nh % cache->nkv == 0, ET_ERR_INVALID_ARG, "et_mha_kv_f16: nh=%d must be a multiple of nkv=%d", nh, cache->nkv);
    const long long width = (long long)nh * cache->hd;
    ET_REQUIRE(ldq >= width && ldz >= width, ET_ERR_INVALID_ARG, "et_mha_kv_f16: row strides %d, %d below nh * hd = %lld", ldq, ldz, width);
    ET_REQUIRE(ldq % 8 == 0 && ldz % 8 == 0, ET_ERR_UNSUPPORTED, "et_mha_kv_f16: row strides must be multiples of 8");
    ET_REQUIRE(((reinterpret_cast<uintptr_t>(Q) | reinterpret_cast<uintptr_t>(Z)) & 15) == 0, ET_ERR_UNSUPPORTED,
               "et_mha_kv_f16: Q and Z must be 16-byte aligned");
    ET_REQUIRE(B <= 65535 && n <= 65535, ET_ERR_UNSUPPORTED, "et_mha_kv_f16: B=%d n=%d", B, n);
    if (B == 0 || n == 0) return ET_OK;
    KvMhaArgs a;
    a.k_codes = static_cast<const unsigned char *>(cache->k_codes);
    a.v_codes = static_cast<const unsigned short *>(cache->v_codes);
    a.k_scales = reinterpret_cast<const unsigned *>(cache->k_scales);
    a.v_scales = reinterpret_cast<const unsigned *>(cache->v_scales);
    a.table = table;
    a.starts = starts;
    a.counts = counts;
    a.Q = reinterpret_cast<const _Float16 *>(Q);
    a.Z = reinterpret_cast<_Float16 *>(Z);
    a.ldq = ldq;
    a.ldz = ldz;
    a.nkv = cache->nkv;
    a.hd = cache->hd;
    a.page = cache->page;
    a.npages = cache->npages;
    a.max_pages = max_pages;
    a.n = n;
    a.nh = nh;
    a.causal = flags & ET_MHA_CAUSAL;
    a.scale_log2e = scale * 1.4426950408889634f;
    return launch_kernel("mha_kv_plain_kernel", cache->bits == 4 ? mha_kv_plain_kernel<4> : mha_kv_plain_kernel<8>, dim3(nh, n, B), 64, 0, as_stream(stream), a);
}

}  // extern "C"
