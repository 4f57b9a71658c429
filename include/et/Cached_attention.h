// Generating token by token (no reference counterpart: its attention sees whole sequences): keys
// and values of every token stay in a paged cache in 4 or 8 bits, and a step runs the new tokens
// alone.  KvCache owns the cache of one layer, KvStep says which tokens a step brings,
// Multihead_attention_cached is the attention, and CachedAttention the block around it: the joined
// Q/K/V projection, the cache written, the attention over it, the output projection.
//
// All launches go to the stream passed to forward(), and nothing in it allocates or blocks, so a
// step can be captured into a HIP graph: table, starts and counts are device memory that the
// caller moves on between replays.
#pragma once
#include <cmath>
#include <memory>
#include <utility>

#include "Linear.h"

namespace et {

// Tokens of one step: rows [b * n, b * n + counts[b]) of the step's matrices are the tokens of
// sequence b from position starts[b] on (counts nullptr: n of each; starts nullptr: from 0).
// table [batch x max_pages]: pages of a sequence, in order.  Device pointers.
struct KvStep {
    const int *table = nullptr;
    int max_pages = 0;
    const int *starts = nullptr;
    const int *counts = nullptr;
    int batch = 1;
    int n = 1;
    bool causal = true;  // a token sees none behind itself (of no concern where n is 1)
};

class KvCache {
  public:
    const int nkv, hd, bits, page, npages;

    KvCache(int _nkv, int _hd, int _bits, int _page, int _npages)
        : nkv(_nkv), hd(_hd), bits(_bits), page(_page), npages(checked(_nkv, _hd, _bits, _page, _npages)),
          k_codes(tokens() * hd * bits / 8), v_codes(tokens() * hd * bits / 8), k_scales(tokens() * (hd / ET_KV_GROUP) * 2),
          v_scales(tokens() * (hd / ET_KV_GROUP) * 2) {}

    et_kv_cache view() const {
        return {k_codes.get(), f16(k_scales.get()), v_codes.get(), f16(v_scales.get()), bits, nkv, hd, page, npages};
    }
    void write(const KvStep &s, const half *k, const half *v, int ldk, int ldv, stream_t stream = nullptr) {
        const et_kv_cache c = view();
        etChk(et_kv_write_f16(&c, s.table, s.max_pages, s.starts, s.counts, f16(k), f16(v), ldk, ldv, s.batch, s.n, stream));
    }
    // the values that the cache stands for; k or v may be nullptr
    void read(const KvStep &s, half *k, half *v, int ldk, int ldv, stream_t stream = nullptr) const {
        const et_kv_cache c = view();
        etChk(et_kv_read_f16(&c, s.table, s.max_pages, s.starts, s.counts, f16(k), f16(v), ldk, ldv, s.batch, s.n, stream));
    }

  private:
    static int checked(int nkv, int hd, int bits, int page, int npages) {
        require(bits == 4 || bits == 8, "KvCache: 4 or 8 bits");
        require(nkv > 0 && npages > 0 && hd > 0 && hd % ET_KV_GROUP == 0 && hd <= 256 && page > 0 && page % 16 == 0,
                "KvCache: heads of a multiple of 32, at most 256, pages of a multiple of 16 tokens");
        return npages;
    }
    std::size_t tokens() const { return (std::size_t)npages * nkv * page; }
    DeviceBuffer<uint8_t> k_codes, v_codes;
    DeviceBuffer<half> k_scales, v_scales;
};

// Device memory that the attention of steps of these sizes, or with fewer pages, needs (0: none).
// Other batches or rows may need more, smaller ones too.
inline std::size_t cached_attention_workspace(const KvCache &cache, int max_pages, int batch, int n, int nhead) {
    const et_kv_cache c = cache.view();
    std::size_t bytes = 0;
    etChk(et_mha_kv_workspace(&c, max_pages, batch, n, nhead, &bytes));
    return bytes;
}

// z = attention of the step's rows over the cache, which holds their own keys and values already.
inline void Multihead_attention_cached(const KvCache &cache, const KvStep &s, const half *q, int ldq, half *z, int ldz, int nhead, void *workspace,
                                       std::size_t workspace_bytes, float scale = 0.0f, stream_t stream = nullptr) {
    const et_kv_cache c = cache.view();
    etChk(et_mha_kv_f16(&c, s.table, s.max_pages, s.starts, s.counts, f16(q), ldq, f16(z), ldz, s.batch, s.n, nhead,
                        scale != 0.0f ? scale : 1.0f / std::sqrt((float)cache.hd), s.causal ? ET_MHA_CAUSAL : 0, workspace, workspace_bytes, stream));
}

// What a Linear's rows have to be a multiple of.
template <typename WEIGHT> constexpr int kLinearRows = 16;
template <> inline constexpr int kLinearRows<w4_mat> = 1;
template <> inline constexpr int kLinearRows<csr_mat> = 1;

// The attention block of a step.  WQKV projects to nhead * hd queries, then nkv * hd keys and
// values; both Linears are made for batch * n rows, a multiple of 16 unless their weights are
// w4_mat or csr_mat.  max_pages: the most that the steps will give.
template <typename WQKV_t, typename WO_t> class CachedAttention {
    std::unique_ptr<Linear<WQKV_t>> linearQKV;
    std::unique_ptr<Linear<WO_t>> linearO;
    std::shared_ptr<KvCache> cache_;
    int nhead, batch, n, max_pages;
    DeviceBuffer<half> qkv, z;
    DeviceBuffer<uint8_t> workspace;

  public:
    CachedAttention(std::unique_ptr<Linear<WQKV_t>> qkv_, std::unique_ptr<Linear<WO_t>> o_, std::shared_ptr<KvCache> cache, int _nhead, int _max_pages, int _batch,
                    int _n = 1)
        : linearQKV(std::move(qkv_)), linearO(std::move(o_)), cache_(checked(std::move(cache), linearQKV && linearO, _batch, _n)), nhead(_nhead), batch(_batch), n(_n), max_pages(_max_pages),
          qkv((std::size_t)_batch * _n * width()), z((std::size_t)_batch * _n * nhead * cache_->hd),
          workspace(cached_attention_workspace(*cache_, _max_pages, _batch, _n, _nhead) + 16) {
        require((int)linearQKV->out_size == width() && (int)linearO->in_size == nhead * cache_->hd && (int)linearQKV->size == batch * n && (int)linearO->size == batch * n,
                "CachedAttention: the projections do not fit the heads, or are made for other rows than batch * n");
    }
    int width() const { return (nhead + 2 * cache_->nkv) * cache_->hd; }
    KvCache &cache() { return *cache_; }
    void forward(half *out, const half *in, const KvStep &s, stream_t stream = nullptr) {
        require(s.batch == batch && s.n == n && s.max_pages <= max_pages, "CachedAttention: a step of other sizes than it was made for");
        const int hd = cache_->hd, ld = width();
        linearQKV->forward(qkv.get(), const_cast<half *>(in), stream);
        cache_->write(s, qkv.get() + nhead * hd, qkv.get() + (nhead + cache_->nkv) * hd, ld, ld, stream);
        Multihead_attention_cached(*cache_, s, qkv.get(), ld, z.get(), nhead * hd, nhead, workspace.get(), workspace.size, 0.0f, stream);
        linearO->forward(out, z.get(), stream);
    }

  private:
    static std::shared_ptr<KvCache> checked(std::shared_ptr<KvCache> cache, bool projections, int batch, int n) {
        require(cache && projections, "CachedAttention: a cache and two projections are needed");
        require(batch > 0 && n > 0, "CachedAttention: batch and n must be at least 1");
        require(batch * n % kLinearRows<WQKV_t> == 0 && batch * n % kLinearRows<WO_t> == 0,
                "CachedAttention: batch * n must be a multiple of 16 for projections other than w4_mat and csr_mat");
        return cache;
    }
};

}  // namespace et
