// What a CachedAttention may be made for and stepped with: tile-sparse projections (16 rows a
// step), fewer pages than it was made for, and what it refuses when it is made.
// Usage: cached_attention_sizes
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>

#include "et/Cached_attention.h"

// values in -1 .. 1, the same on every run
static std::vector<half> values(std::size_t n, uint32_t seed, float size = 1.0f) {
    std::vector<half> v(n);
    uint32_t s = seed * 2654435761u + 1;
    for (auto &x : v) {
        s = s * 1664525u + 1013904223u;
        x = static_cast<half>(size * ((float)(s >> 8) / 8388608.0f - 1.0f));
    }
    return v;
}
static std::vector<float> floats(std::size_t n, uint32_t seed, float size) {
    const auto h = values(n, seed, size);
    std::vector<float> f(n);
    for (std::size_t i = 0; i < n; i++) f[i] = static_cast<float>(h[i]);
    return f;
}
static bool same(const et::DeviceBuffer<half> &a, const et::DeviceBuffer<half> &b) {
    const auto x = a.to_host(), y = b.to_host();
    bool finite = true, zero = true;
    for (half v : x) finite &= std::isfinite((float)v), zero &= (float)v == 0.0f;
    return finite && !zero && x.size() == y.size() && std::memcmp(x.data(), y.data(), x.size() * sizeof(half)) == 0;
}
static int failures = 0;
static void check(bool ok, const char *what) {
    if (!ok) std::printf("FAILED: %s\n", what), failures++;
}
template <typename F> static void refuses(F f, const char *what) {
    bool refused = false;
    try {
        f();
    } catch (const et::Error &) {
        refused = true;
    }
    check(refused, what);
}

static std::vector<int> in_order(int n) {
    std::vector<int> t((std::size_t)n);
    for (int i = 0; i < n; i++) t[(std::size_t)i] = n - 1 - i;
    return t;
}

// Three steps of 16 sequences through tile-sparse projections: what the parts give one after the other.
static void tile_sparse() {
    const int H = 128, nh = 4, nkv = 2, hd = 32, batch = 16, page = 16, max_pages = 2, qkv = (nh + 2 * nkv) * hd;
    auto W = [&](int out, int in, uint32_t seed) {  // every third tile pruned
        auto w = floats((std::size_t)out * in, seed, 0.2f);
        for (int r = 0; r < out; r++)
            for (int c = 0; c < in; c++)
                if ((r / 16 + c / 16) % 3 == 0) w[(std::size_t)r * in + c] = 0.0f;
        return tile_mat::from_dense(w.data(), out, in);
    };
    const auto bq = values(qkv, 3, 0.1f), bo = values(H, 4, 0.1f);
    auto linear = [&](int in, int out, uint32_t seed, const std::vector<half> &b) { return std::make_unique<Linear<tile_mat>>(in, out, W(out, in, seed), b.data(), batch); };
    auto cache = std::make_shared<et::KvCache>(nkv, hd, 4, page, batch * max_pages), own = std::make_shared<et::KvCache>(nkv, hd, 4, page, batch * max_pages);
    et::CachedAttention<tile_mat, tile_mat> block(linear(H, qkv, 1, bq), linear(nh * hd, H, 2, bo), cache, nh, max_pages, batch, 1);
    auto lq = linear(H, qkv, 1, bq), lo = linear(nh * hd, H, 2, bo);
    const et::DeviceBuffer<int> table(in_order(batch * max_pages));
    et::DeviceBuffer<half> y((std::size_t)batch * H), want((std::size_t)batch * H), rows((std::size_t)batch * qkv), z((std::size_t)batch * nh * hd);
    const std::size_t need = et::cached_attention_workspace(*own, max_pages, batch, 1, nh);
    et::DeviceBuffer<uint8_t> ws(need + 16);
    for (int step = 0; step < 3; step++) {
        const et::DeviceBuffer<half> x(values((std::size_t)batch * H, 10 + step));
        const et::DeviceBuffer<int> starts(std::vector<int>((std::size_t)batch, 15 + step));  // over the end of a page
        et::KvStep s;
        s.table = table.get(), s.max_pages = max_pages, s.starts = starts.get(), s.batch = batch, s.n = 1;
        if (step == 0) {
            const et::DeviceBuffer<half> before(values((std::size_t)batch * 15 * nkv * hd, 5));
            et::KvStep b;
            b.table = table.get(), b.max_pages = max_pages, b.batch = batch, b.n = 15;
            for (auto *c : {cache.get(), own.get()}) c->write(b, before.get(), before.get(), nkv * hd, nkv * hd);
        }
        block.forward(y.get(), x.get(), s);
        lq->forward(rows.get(), x.get());
        own->write(s, rows.get() + nh * hd, rows.get() + (nh + nkv) * hd, qkv, qkv);
        et::Multihead_attention_cached(*own, s, rows.get(), qkv, z.get(), nh * hd, nh, ws.get(), need);
        lo->forward(want.get(), z.get());
        etChk(et_device_sync());
        check(same(y, want), "a step with tile-sparse projections");
    }
    refuses([&] { et::CachedAttention<tile_mat, tile_mat>(linear(H, qkv, 1, bq), linear(nh * hd, H, 2, bo), nullptr, nh, max_pages, batch, 1); }, "no cache");
    refuses([&] { et::CachedAttention<tile_mat, tile_mat>(nullptr, linear(nh * hd, H, 2, bo), cache, nh, max_pages, batch, 1); }, "no projection");
    refuses([&] { et::CachedAttention<tile_mat, tile_mat>(linear(H, qkv, 1, bq), nullptr, cache, nh, max_pages, batch, 1); }, "no output projection");
    auto w4 = [&](int in, int out, const std::vector<half> &b, int rows_) {
        return std::make_unique<Linear<w4_mat>>(in, out, w4_mat::from_dense(floats((std::size_t)out * in, 6, 0.2f).data(), out, in, 32), b.data(), rows_);
    };
    auto tile = [&](int in, int out, const std::vector<half> &b, int rows_) { return std::make_unique<Linear<tile_mat>>(in, out, W(out, in, 7), b.data(), rows_); };
    refuses([&] { et::CachedAttention<tile_mat, tile_mat>(tile(H, qkv, bq, 3), tile(nh * hd, H, bo, 3), cache, nh, max_pages, 3, 1); }, "three rows for tile-sparse projections");
    refuses([&] { et::CachedAttention<w4_mat, tile_mat>(w4(H, qkv, bq, 3), tile(nh * hd, H, bo, 3), cache, nh, max_pages, 3, 1); }, "three rows for a tile-sparse output projection");
    et::CachedAttention<w4_mat, w4_mat> three(w4(H, qkv, bq, 3), w4(nh * hd, H, bo, 3), cache, nh, max_pages, 3, 1);
    check(three.width() == qkv, "three rows for 4-bit projections");
}

// Made for 128 pages and stepped with 127: as if made for those.
static void fewer_pages() {
    const int H = 64, nh = 64, nkv = 8, hd = 128, batch = 4, page = 16, most = 128, pages = 127, qkv = (nh + 2 * nkv) * hd;
    auto cache = std::make_shared<et::KvCache>(nkv, hd, 4, page, batch * most);
    const w4_mat wq = w4_mat::from_dense(floats((std::size_t)qkv * H, 1, 0.2f).data(), qkv, H), wo = w4_mat::from_dense(floats((std::size_t)nh * hd * H, 2, 0.02f).data(), H, nh * hd);
    const auto bq = values(qkv, 3, 0.1f), bo = values(H, 4, 0.1f);
    auto block = [&](int p) {
        return std::make_unique<et::CachedAttention<w4_mat, w4_mat>>(std::make_unique<Linear<w4_mat>>(H, qkv, wq, bq.data(), batch),
                                                                    std::make_unique<Linear<w4_mat>>(nh * hd, H, wo, bo.data(), batch), cache, nh, p, batch, 1);
    };
    const et::DeviceBuffer<int> table(in_order(batch * pages)), starts(std::vector<int>{2000, 2031, 7, 1024});
    const et::DeviceBuffer<half> before(values((std::size_t)batch * 2031 * nkv * hd, 5)), x(values((std::size_t)batch * H, 6));
    et::KvStep b;
    b.table = table.get(), b.max_pages = pages, b.batch = batch, b.n = 2031;
    cache->write(b, before.get(), before.get(), nkv * hd, nkv * hd);
    et::KvStep s;
    s.table = table.get(), s.max_pages = pages, s.starts = starts.get(), s.batch = batch, s.n = 1;
    et::DeviceBuffer<half> y((std::size_t)batch * H), want((std::size_t)batch * H);
    block(most)->forward(y.get(), x.get(), s);
    block(pages)->forward(want.get(), x.get(), s);
    etChk(et_device_sync());
    check(same(y, want), "fewer pages than it was made for");
}

int main() {
    try {
        tile_sparse();
        fewer_pages();
    } catch (const std::exception &e) {
        std::fprintf(stderr, "%s\n", e.what());
        return 1;
    }
    if (failures == 0) std::printf("ok\n");
    return failures ? 1 : 0;
}
