// Attention over a cache of keys and values in 4 or 8 bits, whose rows see a window and the first tokens, or the nodes of a tree.
//
// A block of rows walks over the tiles that some of its rows see, those of the first tokens and from the earliest window on: pages in between are neither read nor looked up.  Keys are masked
// one by one only in tiles that are not seen whole: at a window's beginning, at the end, and where the tree's own tokens lie, whose 32 bits a row and tile are two words of it.
#include "attention_kv_tile.h"

namespace et {
namespace {

// Positions that the rows of a block see at most, rounded up by a tile at either end.  (Rows that see what stands behind them see up to n more: their keys are shared out as those of rows
// that do not, so that a workspace needs no flags.)
long long sight_positions(const et_kv_cache *cache, int max_pages, int n, int nh, int window, int sinks) {
    const long long all = (long long)max_pages * cache->page, apart = std::max(16, 256 / std::max(1, nh / cache->nkv));
    return window == 0 ? all : std::min(all, (long long)window + sinks + std::min((long long)n, apart) + 128);
}

int check_window(const char *fn, int window, int sinks, int least) {
    ET_REQUIRE(window >= least && sinks >= 0, ET_ERR_INVALID_ARG, "%s: window=%d sinks=%d, the window must be at least %d", fn, window, sinks, least);
    return ET_OK;
}

constexpr int kMostNodes = 256;

int check_tree(const char *fn, int n, int window, int sinks) {
    ET_REQUIRE(n <= kMostNodes, ET_ERR_UNSUPPORTED, "%s: n=%d, a tree has up to %d tokens", fn, n, kMostNodes);
    // (a node must not lose sight of one on its way up)
    return check_window(fn, window, sinks, window == 0 ? 0 : n);
}

// Rows of a key/value head in the call.
long long rows_of(const et_kv_cache *cache, int n, int nh) { return (long long)n * std::max(0, nh / cache->nkv); }

// (The larger of what both kinds of kernel need where the rows are many: which of them runs depends on the positions, and a workspace is to do for fewer pages, too.)
int sight_workspace(const char *fn, const et_kv_cache *cache, int max_pages, int B, int n, int nh, int window, int sinks, size_t *bytes) {
    const long long positions = sight_positions(cache, max_pages, n, nh, window, sinks);
    KvPlan<true> p;
    int st = kv_plan<true>(fn, p, cache, positions, B, n, nh);
    if (st != ET_OK) return st;
    KvTilePlan tile;
    tile.bytes = 0;
    const int waves = kv_tile_most_waves(cache->hd, rows_of(cache, n, nh));
    if (waves) st = kv_tile_plan(fn, tile, cache, positions, B, n, nh, waves);
    if (st == ET_OK) *bytes = std::max(p.bytes, tile.bytes);
    return st;
}

int sight_run(const char *fn, const KvMhaCall &call, KvSightArgs &a, et_stream stream) {
    const long long positions = sight_positions(call.cache, call.max_pages, call.n, call.nh, a.window, a.sinks), rows = rows_of(call.cache, call.n, call.nh);
    size_t need = 0;
    const int st = sight_workspace(fn, call.cache, call.max_pages, call.B, call.n, call.nh, a.window, a.sinks, &need);
    if (st != ET_OK) return st;
    const int waves = kv_tile_waves(call.cache, positions, call.B, rows);
    if (waves) return kv_tile_run(fn, call, positions, waves, need, a, stream);
    return kv_run<true>(fn, call, positions, need, a, stream);
}

}  // namespace
}  // namespace et

using namespace et;

extern "C" {

int et_mha_kv_window_workspace(const et_kv_cache *cache, int max_pages, int B, int n, int nh, int window, int sinks, size_t *bytes) {
    static const char *fn = "et_mha_kv_window_workspace";
    ET_REQUIRE(bytes, ET_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    static const int32_t any = 0;
    int st = kv_check_cache(fn, cache, &any, max_pages, B, n);
    if (st == ET_OK) st = check_window(fn, window, sinks, 1);
    return st != ET_OK ? st : sight_workspace(fn, cache, max_pages, B, n, nh, window, sinks, bytes);
}

int et_mha_kv_window_f16(const et_kv_cache *cache, const int32_t *table, int max_pages, const int32_t *starts, const int32_t *counts, const et_f16 *Q, int ldq,
                         et_f16 *Z, int ldz, int B, int n, int nh, int window, int sinks, float scale, int flags, void *workspace, size_t workspace_bytes,
                         et_stream stream) {
    static const char *fn = "et_mha_kv_window_f16";
    ET_REQUIRE(Q && Z, ET_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    int st = kv_check_cache(fn, cache, table, max_pages, B, n);
    if (st == ET_OK) st = check_window(fn, window, sinks, 1);
    if (st != ET_OK) return st;
    ET_REQUIRE((flags & ~ET_MHA_CAUSAL) == 0, ET_ERR_INVALID_ARG, "%s: flags=%d", fn, flags);
    KvSightArgs a;
    a.causal = flags & ET_MHA_CAUSAL;
    a.window = window;
    a.sinks = sinks;
    a.seen = nullptr;
    a.words = 0;
    return sight_run(fn, {cache, table, max_pages, starts, counts, Q, ldq, Z, ldz, B, n, nh, scale, workspace, workspace_bytes}, a, stream);
}

int et_mha_kv_tree_workspace(const et_kv_cache *cache, int max_pages, int B, int n, int nh, int window, int sinks, size_t *bytes) {
    static const char *fn = "et_mha_kv_tree_workspace";
    ET_REQUIRE(bytes, ET_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    static const int32_t any = 0;
    int st = kv_check_cache(fn, cache, &any, max_pages, B, n);
    if (st == ET_OK) st = check_tree(fn, n, window, sinks);
    return st != ET_OK ? st : sight_workspace(fn, cache, max_pages, B, n, nh, window, sinks, bytes);
}

int et_mha_kv_tree_f16(const et_kv_cache *cache, const int32_t *table, int max_pages, const int32_t *starts, const int32_t *counts, const uint32_t *seen,
                       const et_f16 *Q, int ldq, et_f16 *Z, int ldz, int B, int n, int nh, int window, int sinks, float scale, void *workspace,
                       size_t workspace_bytes, et_stream stream) {
    static const char *fn = "et_mha_kv_tree_f16";
    ET_REQUIRE(Q && Z && seen, ET_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    int st = kv_check_cache(fn, cache, table, max_pages, B, n);
    if (st == ET_OK) st = check_tree(fn, n, window, sinks);
    if (st != ET_OK) return st;
    ET_REQUIRE((reinterpret_cast<uintptr_t>(seen) & 3) == 0, ET_ERR_UNSUPPORTED, "%s: seen must be 4-byte aligned", fn);
    KvSightArgs a;
    a.causal = 0;
    a.window = window;
    a.sinks = sinks;
    a.seen = seen;
    a.words = (n + 31) / 32;
    return sight_run(fn, {cache, table, max_pages, starts, counts, Q, ldq, Z, ldz, B, n, nh, scale, workspace, workspace_bytes}, a, stream);
}

}  // extern "C"
