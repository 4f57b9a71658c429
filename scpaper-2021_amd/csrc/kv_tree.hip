// Trees of guessed tokens behind the sequences of a cache: which nodes a node sees, the path that the model itself chose, and the cache moved together over it (et_abi.h).
//
// All three are a few dependent accesses on a few kilobytes, and bound by a launch and those: 8 sequences of 16 nodes take 2.0 us for what they see, 3.4 for the path and 4.2 for 12 heads of 64
// moved.  With 64 sequences of 64 nodes the path takes 3.7 us, and six layers of 16 heads of 64 in 8 bits 20: of the values a token is 2 of every 8 bytes, so that four times what is moved is
// read and written.
#include "common.hip.h"

namespace et {

int kv_check_cache(const char *fn, const et_kv_cache *c, const int32_t *table, int max_pages, int B, int n);

namespace {

constexpr int kMostNodes = 256;

__device__ __forceinline__ int tree_count(const int32_t *counts, int b, int n) { return counts ? min(max(counts[b], 0), n) : n; }

// A node's bits are its own and those of the nodes on its way up.  Each round a node takes over the bits of the one that its pointer has come to, and that one's pointer: ways of
// length 2^r are done after r rounds, where a walk up takes as many dependent steps as the tree is deep.
template <int W> __global__ __launch_bounds__(32 * W < 64 ? 64 : 32 * W) void tree_seen_kernel(const int32_t *parents, const int32_t *counts, unsigned *seen, int n) {
    __shared__ unsigned bits[2][W][32 * W];
    __shared__ int up[2][32 * W];
    const int b = blockIdx.x, i = threadIdx.x, words = (n + 31) / 32;
    const int count = tree_count(counts, b, n);
    const int p = parents[(size_t)b * n + min(i, n - 1)];  // (asked for without waiting for the count)
    const bool there = i < count;
    int at = there && p >= 0 && p < i ? p : -1;
    unsigned own[W];
#pragma unroll
    for (int w = 0; w < W; w++) own[w] = i >> 5 == w ? 1u << (i & 31) : 0u;
    for (int side = 0; __syncthreads_or(at >= 0); side ^= 1) {
        if (i < 32 * W) {
#pragma unroll
            for (int w = 0; w < W; w++) bits[side][w][i] = own[w];
            up[side][i] = at;
        }
        __syncthreads();
        if (at >= 0) {
#pragma unroll
            for (int w = 0; w < W; w++) own[w] |= bits[side][w][at];
            at = up[side][at];
        }
    }
    if (there) {
        unsigned *to = seen + ((size_t)b * n + i) * words;
#pragma unroll
        for (int w = 0; w < W; w++)
            if (w < words) to[w] = own[w];
    }
}

// One wave a sequence, up to four nodes a lane: each step asks all of them at once whose parent is the current node and whose token is the one chosen after it.
__global__ __launch_bounds__(64) void tree_follow_kernel(const int32_t *parents, const int32_t *tokens, const int32_t *choices, const int32_t *starts, const int32_t *counts,
                                                         int32_t *path, int32_t *kept, int32_t *next_tokens, int32_t *next_starts, int n) {
    constexpr int K = kMostNodes / 64;
    __shared__ int chosen[kMostNodes], way[kMostNodes];
    const int b = blockIdx.x, lane = threadIdx.x;
    const int start = starts ? starts[b] : 0, count = tree_count(counts, b, n);
    int parent[K], token[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int i = lane + 64 * k;
        const size_t at = (size_t)b * n + min(i, n - 1);
        const int p = parents[at], t = tokens[at], c = choices[at];
        parent[k] = i < count ? p : -1;
        token[k] = t;
        chosen[i] = c;
        way[i] = -1;
    }
    wave_lds_order();
    int now = count > 0 ? 0 : -1, steps = 0, next = -1;
    while (now >= 0) {
        if (lane == 0) way[steps] = now;
        steps++;
        next = chosen[now];
        int child = -1;
#pragma unroll
        for (int k = 0; k < K; k++) {
            // (a node's parent stands before it: what says otherwise has none, and the way ends after n nodes at most)
            const unsigned long long fit = __ballot(parent[k] == now && token[k] == next && lane + 64 * k > now);
            if (child < 0 && fit != 0) child = 64 * k + __builtin_ctzll(fit);
        }
        now = __builtin_amdgcn_readfirstlane(child);
    }
    wave_lds_order();
    for (int i = lane; i < n; i += 64) path[(size_t)b * n + i] = way[i];
    if (lane == 0) {
        kept[b] = steps;
        next_tokens[b] = next;
        next_starts[b] = (int)min((long long)start + steps, 0x7fffffffLL);
    }
}

constexpr int kKeepCaches = 64;

struct KeepArgs {
    struct {
        char *k_codes, *v_codes;
        unsigned *k_scales, *v_scales;
    } of[kKeepCaches];
    const int32_t *table, *starts, *path, *kept;
    int max_pages, n, nkv, hd, page, npages;
    int rows_log2;  // threads of a (head, group): rows up to n
};

// A thread moves one row's 32 channels of a head, keys and values: all threads of a (head, group) read before any of them writes, so that rows may come from any place.
template <int BITS> __global__ __launch_bounds__(256) void kv_keep_kernel(const KeepArgs a) {
    constexpr int Q = BITS / 4, U = 2 * BITS;  // 16-byte pieces of a key, units of 16 bits of a value
    const int b = blockIdx.y, groups = a.hd / ET_KV_GROUP;
    const int r = threadIdx.x & ((1 << a.rows_log2) - 1), unit = (int)(blockIdx.x << (8 - a.rows_log2)) + (int)(threadIdx.x >> a.rows_log2);
    const auto &cache = a.of[blockIdx.z];
    const int kept = min(max(a.kept[b], 0), a.n);
    const long long start = a.starts ? a.starts[b] : 0;
    const int from_row = r < a.n ? a.path[(size_t)b * a.n + r] : -1;
    // a position's token, counted [pages][nkv][page], or -1
    struct Place { long long page; int off; };
    auto place = [&](long long pos) {
        const long long page_at = pos / a.page;
        const int page = pos >= 0 && page_at < a.max_pages ? a.table[(size_t)b * a.max_pages + page_at] : -1;
        return Place{page >= 0 && page < a.npages ? page : -1, (int)(pos - page_at * a.page)};
    };
    const int head = unit / groups, group = unit - head * groups;
    bool moves = r < kept && unit < a.nkv * groups && from_row >= 0 && from_row < a.n && from_row != r;
    Place from{-1, 0}, to{-1, 0};
    if (moves) {
        from = place(start + from_row);
        to = place(start + r);
        moves = from.page >= 0 && to.page >= 0;
    }
    const int token_bytes = a.hd * BITS / 8;
    uint4 key[Q];
    unsigned short value[U];
    unsigned k_scale = 0, v_scale = 0;
    auto key_at = [&](Place p) { return cache.k_codes + ((size_t)(p.page * a.nkv + head) * a.page + p.off) * token_bytes + group * (4 * BITS); };
    auto value_at = [&](Place p) { return cache.v_codes + ((size_t)(p.page * a.nkv + head) * a.page + (p.off & ~3)) * token_bytes + group * (16 * BITS) + (p.off & 3) * 2; };
    auto scale_at = [&](Place p) { return ((size_t)(p.page * a.nkv + head) * groups + group) * a.page + p.off; };
    if (moves) {
#pragma unroll
        for (int i = 0; i < Q; i++) key[i] = *reinterpret_cast<const uint4 *>(key_at(from) + 16 * i);
#pragma unroll
        for (int i = 0; i < U; i++) value[i] = *reinterpret_cast<const unsigned short *>(value_at(from) + 8 * i);
        k_scale = cache.k_scales[scale_at(from)];
        v_scale = cache.v_scales[scale_at(from)];
    }
    __syncthreads();
    if (!moves) return;
#pragma unroll
    for (int i = 0; i < Q; i++) *reinterpret_cast<uint4 *>(key_at(to) + 16 * i) = key[i];
#pragma unroll
    for (int i = 0; i < U; i++) *reinterpret_cast<unsigned short *>(value_at(to) + 8 * i) = value[i];
    cache.k_scales[scale_at(to)] = k_scale;
    cache.v_scales[scale_at(to)] = v_scale;
}

int check_tree(const char *fn, int B, int n) {
    ET_REQUIRE(B >= 0 && n >= 0, ET_ERR_INVALID_ARG, "%s: B=%d n=%d", fn, B, n);
    ET_REQUIRE(B <= 65535 && n <= kMostNodes, ET_ERR_UNSUPPORTED, "%s: B=%d n=%d, a tree has up to %d tokens", fn, B, n, kMostNodes);
    return ET_OK;
}

}  // namespace
}  // namespace et

using namespace et;

extern "C" {

int et_tree_seen(const int32_t *parents, const int32_t *counts, uint32_t *seen, int B, int n, et_stream stream) {
    ET_REQUIRE(parents && seen, ET_ERR_INVALID_ARG, "et_tree_seen: NULL pointer");
    const int st = check_tree("et_tree_seen", B, n);
    if (st != ET_OK || B == 0 || n == 0) return st;
    ET_REQUIRE(((reinterpret_cast<uintptr_t>(parents) | reinterpret_cast<uintptr_t>(counts) | reinterpret_cast<uintptr_t>(seen)) & 3) == 0, ET_ERR_UNSUPPORTED,
               "et_tree_seen: arrays must be 4-byte aligned");
    const int words = (n + 31) / 32;
    return launch_kernel("tree_seen_kernel", words == 1 ? tree_seen_kernel<1> : words == 2 ? tree_seen_kernel<2> : words <= 4 ? tree_seen_kernel<4> : tree_seen_kernel<8>, dim3((unsigned)B),
                         words <= 2 ? 64 : words <= 4 ? 128 : 256, 0, as_stream(stream), parents, counts, seen, n);
}

int et_tree_follow(const int32_t *parents, const int32_t *tokens, const int32_t *choices, const int32_t *starts, const int32_t *counts, int32_t *path, int32_t *kept,
                   int32_t *next_tokens, int32_t *next_starts, int B, int n, et_stream stream) {
    ET_REQUIRE(parents && tokens && choices && path && kept && next_tokens && next_starts, ET_ERR_INVALID_ARG, "et_tree_follow: NULL pointer");
    const int st = check_tree("et_tree_follow", B, n);
    if (st != ET_OK) return st;
    ET_REQUIRE(n > 0, ET_ERR_INVALID_ARG, "et_tree_follow: n=%d", n);
    if (B == 0) return ET_OK;
    return launch_kernel("tree_follow_kernel", tree_follow_kernel, dim3((unsigned)B), 64, 0, as_stream(stream), parents, tokens, choices, starts, counts, path, kept, next_tokens,
                         next_starts, n);
}

int et_kv_keep(const et_kv_cache *caches, int ncaches, const int32_t *table, int max_pages, const int32_t *starts, const int32_t *path, const int32_t *kept, int B, int n,
               et_stream stream) {
    ET_REQUIRE(caches && ncaches > 0 && path && kept, ET_ERR_INVALID_ARG, "et_kv_keep: NULL pointer, or ncaches=%d", ncaches);
    const et_kv_cache &first = caches[0];
    for (int i = 0; i < ncaches; i++) {
        const et_kv_cache &c = caches[i];
        const int st = kv_check_cache("et_kv_keep", &c, table, max_pages, B, n);
        if (st != ET_OK) return st;
        ET_REQUIRE(c.bits == first.bits && c.nkv == first.nkv && c.hd == first.hd && c.page == first.page && c.npages == first.npages, ET_ERR_INVALID_ARG,
                   "et_kv_keep: cache %d has other sizes than the first", i);
    }
    const int st = check_tree("et_kv_keep", B, n);
    if (st != ET_OK || B == 0 || n == 0) return st;
    // (moved twice at once, what one has written the other would read)
    for (int i = 1; i < ncaches; i++)
        for (int j = 0; j < i; j++)
            ET_REQUIRE(caches[i].k_codes != caches[j].k_codes && caches[i].v_codes != caches[j].v_codes && caches[i].k_scales != caches[j].k_scales &&
                           caches[i].v_scales != caches[j].v_scales, ET_ERR_INVALID_ARG, "et_kv_keep: caches %d and %d are the same", j, i);
    KeepArgs a;
    a.table = table;
    a.starts = starts;
    a.path = path;
    a.kept = kept;
    a.max_pages = max_pages;
    a.n = n;
    a.nkv = first.nkv;
    a.hd = first.hd;
    a.page = first.page;
    a.npages = first.npages;
    a.rows_log2 = 0;
    while ((1 << a.rows_log2) < n) a.rows_log2++;
    const unsigned units = (unsigned)(first.nkv * (first.hd / ET_KV_GROUP)), of_workgroup = 256u >> a.rows_log2;
    for (int at = 0; at < ncaches; at += kKeepCaches) {
        const int some = ncaches - at < kKeepCaches ? ncaches - at : kKeepCaches;
        for (int i = 0; i < kKeepCaches; i++) {
            const et_kv_cache &c = caches[at + (i < some ? i : 0)];
            a.of[i] = {static_cast<char *>(c.k_codes), static_cast<char *>(c.v_codes), reinterpret_cast<unsigned *>(c.k_scales), reinterpret_cast<unsigned *>(c.v_scales)};
        }
        const int sl = launch_kernel("kv_keep_kernel", first.bits == 4 ? kv_keep_kernel<4> : kv_keep_kernel<8>, dim3((units + of_workgroup - 1) / of_workgroup, (unsigned)B, (unsigned)some), 256,
                                     0, as_stream(stream), a);
        if (sl != ET_OK) return sl;
    }
    return ET_OK;
}

}  // extern "C"
