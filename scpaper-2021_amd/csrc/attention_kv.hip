// Attention over a cache of keys and values in 4 or 8 bits, whose rows see all keys or those up to their own; joining the parts of keys that are shared out.
#include "attention_kv.hip.h"

namespace et {

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

int kv_join(const KvMhaArgs &a, int blocks, hipStream_t stream) {
    const int lots_log2 = a.splits <= 4 ? 0 : a.splits <= 8 ? 1 : a.splits <= 16 ? 2 : 3;
    const int channels = a.units * a.block_rows * (a.hd / ET_KV_GROUP), of_workgroup = 8 >> lots_log2;
    return launch_kernel("mha_kv_join_kernel", mha_kv_join_kernel, dim3((unsigned)((channels + of_workgroup - 1) / of_workgroup), (unsigned)blocks), 256, 0, stream, a, lots_log2);
}

}  // namespace et

using namespace et;

extern "C" {

int et_mha_kv_workspace(const et_kv_cache *cache, int max_pages, int B, int n, int nh, size_t *bytes) {
    ET_REQUIRE(bytes, ET_ERR_INVALID_ARG, "et_mha_kv_workspace: NULL pointer");
    static const int32_t any = 0;
    const int st = kv_check_cache("et_mha_kv_workspace", cache, &any, max_pages, B, n);
    if (st != ET_OK) return st;
    KvPlan<false> p;
    const int sp = kv_plan<false>("et_mha_kv_workspace", p, cache, (long long)max_pages * cache->page, B, n, nh);
    if (sp == ET_OK) *bytes = p.bytes;
    return sp;
}

int et_mha_kv_f16(const et_kv_cache *cache, const int32_t *table, int max_pages, const int32_t *starts, const int32_t *counts, const et_f16 *Q, int ldq,
                  et_f16 *Z, int ldz, int B, int n, int nh, float scale, int flags, void *workspace, size_t workspace_bytes, et_stream stream) {
    ET_REQUIRE(Q && Z, ET_ERR_INVALID_ARG, "et_mha_kv_f16: NULL pointer");
    const int st = kv_check_cache("et_mha_kv_f16", cache, table, max_pages, B, n);
    if (st != ET_OK) return st;
    ET_REQUIRE((flags & ~ET_MHA_CAUSAL) == 0, ET_ERR_INVALID_ARG, "et_mha_kv_f16: flags=%d", flags);
    KvMhaArgs a;
    a.causal = flags & ET_MHA_CAUSAL;
    return kv_run<false>("et_mha_kv_f16", {cache, table, max_pages, starts, counts, Q, ldq, Z, ldz, B, n, nh, scale, workspace, workspace_bytes}, (long long)max_pages * cache->page, 0, a, stream);
}

}  // extern "C"
