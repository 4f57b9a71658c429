// Generating token by token (no reference counterpart: its attention sees whole sequences): keys
// and values of every token stay in a paged cache in 4 or 8 bits, and a step runs the new tokens
// alone.  KvCache owns the cache of one layer, KvStep says which tokens a step brings,
// Multihead_attention_cached is the attention, and CachedAttention the block around it: the joined
// Q/K/V projection, the cache written, the attention over it, the output projection.  KvPages hands
// out a cache's pages on the device, and GuessedTokens is a step's tree of guessed tokens.
//
// All launches go to the stream passed to forward(), and nothing in it allocates or blocks, so a
// step can be captured into a HIP graph: table, starts and counts are device memory that the
// caller moves on between replays.
#pragma once
#include <algorithm>
#include <cmath>
#include <memory>
#include <utility>
#include <vector>

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
    int window = 0;      // tokens that a token sees, itself the last, and the first `sinks` of the sequence; 0: all
    int sinks = 0;
    const uint32_t *seen = nullptr;  // the rows are nodes of trees (GuessedTokens::see): what each sees of the others; causal is of no concern
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
// Other batches or rows may need more, smaller ones too.  window, sinks, tree: of steps that have
// them.
inline std::size_t cached_attention_workspace(const KvCache &cache, int max_pages, int batch, int n, int nhead, int window = 0, int sinks = 0, bool tree = false) {
    const et_kv_cache c = cache.view();
    std::size_t bytes = 0;
    if (tree)
        etChk(et_mha_kv_tree_workspace(&c, max_pages, batch, n, nhead, window, sinks, &bytes));
    else if (window != 0)
        etChk(et_mha_kv_window_workspace(&c, max_pages, batch, n, nhead, window, sinks, &bytes));
    else
        etChk(et_mha_kv_workspace(&c, max_pages, batch, n, nhead, &bytes));
    return bytes;
}

// z = attention of the step's rows over the cache, which holds their own keys and values already.
inline void Multihead_attention_cached(const KvCache &cache, const KvStep &s, const half *q, int ldq, half *z, int ldz, int nhead, void *workspace,
                                       std::size_t workspace_bytes, float scale = 0.0f, stream_t stream = nullptr) {
    const et_kv_cache c = cache.view();
    const float by = scale != 0.0f ? scale : 1.0f / std::sqrt((float)cache.hd);
    const int flags = s.causal ? ET_MHA_CAUSAL : 0;
    if (s.seen)
        etChk(et_mha_kv_tree_f16(&c, s.table, s.max_pages, s.starts, s.counts, s.seen, f16(q), ldq, f16(z), ldz, s.batch, s.n, nhead, s.window, s.sinks, by, workspace, workspace_bytes,
                                 stream));
    else if (s.window != 0)
        etChk(et_mha_kv_window_f16(&c, s.table, s.max_pages, s.starts, s.counts, f16(q), ldq, f16(z), ldz, s.batch, s.n, nhead, s.window, s.sinks, by, flags, workspace, workspace_bytes,
                                   stream));
    else
        etChk(et_mha_kv_f16(&c, s.table, s.max_pages, s.starts, s.counts, f16(q), ldq, f16(z), ldz, s.batch, s.n, nhead, by, flags, workspace, workspace_bytes, stream));
}

// The pages of a cache, handed out on the device: a table [batch x max_pages], which the layers of a
// model share, and the free pages.  give() makes a step's table hold pages for what its rows see,
// and takes back those that no row sees any more (behind a window, or of a sequence that is over:
// start and count 0).  One step at a time: launches of give() must not overlap.
class KvPages {
  public:
    const int batch, max_pages, page, npages;

    KvPages(const KvCache &cache, int _batch, int _max_pages)
        : batch(_batch), max_pages(_max_pages), page(cache.page), npages(cache.npages), table_(std::vector<int>(checked(_batch, _max_pages), -1)), free_(numbers(cache.npages)),
          state_(std::vector<int>{0, cache.npages, 0}), workspace(needed(_batch, _max_pages) + 16) {}

    // s.table and s.max_pages become this table.  slots [batch][n], 8 bytes each: where each row lies
    // (page * the page's tokens + its place), or -1; shared [batch]: so many entries of a sequence
    // stay as they are.
    void give(KvStep &s, int64_t *slots = nullptr, const int *shared = nullptr, stream_t stream = nullptr) {
        require(s.batch == batch, "KvPages: a step of another batch");
        s.table = table_.get(), s.max_pages = max_pages;
        etChk(et_kv_tables(table_.get(), table_.get(), max_pages, page, npages, s.starts, s.counts, shared, batch, s.n, s.window, s.sinks, free_.get(), state_.get(), state_.get(), slots,
                           workspace.get(), workspace.size, stream));
    }
    int *table() { return table_.get(); }
    // of the last step, once the device has done it
    int free_pages() const { return state_.to_host()[1]; }
    int missing() const { return state_.to_host()[2]; }

  private:
    static std::size_t checked(int batch, int max_pages) {
        require(batch > 0 && max_pages > 0, "KvPages: batch and pages must be at least 1");
        return (std::size_t)batch * max_pages;
    }
    static std::vector<int> numbers(int n) {
        std::vector<int> v((std::size_t)n);
        for (int i = 0; i < n; i++) v[(std::size_t)i] = i;
        return v;
    }
    static std::size_t needed(int batch, int max_pages) {
        std::size_t bytes = 0;
        etChk(et_kv_tables_workspace(max_pages, batch, &bytes));
        return bytes;
    }
    DeviceBuffer<int> table_, free_, state_;
    DeviceBuffer<uint8_t> workspace;
};

// A tree of up to n guessed tokens for each sequence: node 0 is the token that the model chose last,
// and follows on the cache's last position.  Of a step: see(), then the layers with s.seen, then
// follow() with what the model chose after each node, and keep() with each layer's cache.
class GuessedTokens {
  public:
    const int batch, n;
    DeviceBuffer<uint32_t> seen;
    DeviceBuffer<int> path, kept;  // [batch x n], the nodes that stand, then -1; [batch], how many

    GuessedTokens(int _batch, int _n) : batch(_batch), n(_n), seen(checked(_batch, _n)), path((std::size_t)_batch * _n), kept((std::size_t)_batch) {}

    // parents [batch x n]: a smaller number each, node 0's is -1
    void see(KvStep &s, const int *parents, stream_t stream = nullptr) {
        require(s.batch == batch && s.n == n, "GuessedTokens: a step of other sizes");
        etChk(et_tree_seen(parents, s.counts, seen.get(), batch, n, stream));
        s.seen = seen.get();
    }
    // tokens, choices [batch x n]: each node's token, and what the model chose after it.  next_tokens,
    // next_starts [batch]: node 0 of the next step, and its position (not s.starts, which keep() reads)
    void follow(const KvStep &s, const int *parents, const int *tokens, const int *choices, int *next_tokens, int *next_starts, stream_t stream = nullptr) {
        require(s.batch == batch && s.n == n, "GuessedTokens: a step of other sizes");
        require(next_starts != s.starts, "GuessedTokens: the step's starts are still needed");
        etChk(et_tree_follow(parents, tokens, choices, s.starts, s.counts, path.get(), kept.get(), next_tokens, next_starts, batch, n, stream));
    }
    // the tokens that stand, moved together in the caches of the layers
    void keep(const KvStep &s, const std::vector<const KvCache *> &caches, stream_t stream = nullptr) {
        require(s.batch == batch && s.n == n && !caches.empty(), "GuessedTokens: a step of other sizes, or no cache");
        std::vector<et_kv_cache> views;
        for (const KvCache *c : caches) views.push_back(c->view());
        etChk(et_kv_keep(views.data(), (int)views.size(), s.table, s.max_pages, s.starts, path.get(), kept.get(), batch, n, stream));
    }

  private:
    static std::size_t checked(int batch, int n) {
        require(batch > 0 && n > 0 && n <= 256, "GuessedTokens: 1 to 256 tokens for at least one sequence");
        return (std::size_t)batch * n * ((n + 31) / 32);
    }
};

// What a Linear's rows have to be a multiple of.
template <typename WEIGHT> constexpr int kLinearRows = 16;
template <> inline constexpr int kLinearRows<w4_mat> = 1;
template <> inline constexpr int kLinearRows<csr_mat> = 1;

// The attention block of a step.  WQKV projects to nhead * hd queries, then nkv * hd keys and
// values; both Linears are made for batch * n rows, a multiple of 16 unless their weights are
// w4_mat or csr_mat.  max_pages: the most that the steps will give; window, sinks: those of every
// step; tree: steps may bring trees, with or without a window.
template <typename WQKV_t, typename WO_t> class CachedAttention {
    std::unique_ptr<Linear<WQKV_t>> linearQKV;
    std::unique_ptr<Linear<WO_t>> linearO;
    std::shared_ptr<KvCache> cache_;
    int nhead, batch, n, max_pages, window, sinks;
    bool tree;
    DeviceBuffer<half> qkv, z;
    DeviceBuffer<uint8_t> workspace;

  public:
    CachedAttention(std::unique_ptr<Linear<WQKV_t>> qkv_, std::unique_ptr<Linear<WO_t>> o_, std::shared_ptr<KvCache> cache, int _nhead, int _max_pages, int _batch,
                    int _n = 1, int _window = 0, int _sinks = 0, bool _tree = false)
        : linearQKV(std::move(qkv_)), linearO(std::move(o_)), cache_(checked(std::move(cache), linearQKV && linearO, _batch, _n)), nhead(_nhead), batch(_batch), n(_n), max_pages(_max_pages),
          window(_window), sinks(_sinks), tree(_tree), qkv((std::size_t)_batch * _n * width()), z((std::size_t)_batch * _n * nhead * cache_->hd),
          workspace(std::max(cached_attention_workspace(*cache_, _max_pages, _batch, _n, _nhead, _window, _sinks),
                             _tree ? cached_attention_workspace(*cache_, _max_pages, _batch, _n, _nhead, _window, _sinks, true) : 0) + 16) {
        require((int)linearQKV->out_size == width() && (int)linearO->in_size == nhead * cache_->hd && (int)linearQKV->size == batch * n && (int)linearO->size == batch * n,
                "CachedAttention: the projections do not fit the heads, or are made for other rows than batch * n");
    }
    int width() const { return (nhead + 2 * cache_->nkv) * cache_->hd; }
    KvCache &cache() { return *cache_; }
    void forward(half *out, const half *in, const KvStep &s, stream_t stream = nullptr) {
        require(s.batch == batch && s.n == n && s.max_pages <= max_pages, "CachedAttention: a step of other sizes than it was made for");
        require(s.window == window && s.sinks == sinks && (tree || !s.seen), "CachedAttention: a step of another window, or a tree, than it was made for");
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
