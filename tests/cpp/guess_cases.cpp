// Guessing several tokens at once through the C++ class layer: pages handed out on the device, two
// CachedAttention blocks over trees with a window, the path that stands and what stands moved
// together, recorded in a graph once and replayed; results written as .npy files for the Python
// side to compare.  Before that, what the classes refuse.
// Usage: guess_cases <dir>
#include <cstdio>
#include <string>

#include "et/Cached_attention.h"
#include "et/npy.hpp"

using et::npy::npy_load;
using et::npy::npy_save;

static std::vector<half> as_half(const std::vector<float> &f) {
    std::vector<half> h(f.size());
    for (std::size_t i = 0; i < f.size(); i++) h[i] = static_cast<half>(f[i]);
    return h;
}
template <typename F> static bool refuses(F f) {
    try {
        f();
    } catch (const et::Error &) {
        return true;
    }
    return false;
}

int main(int argc, char **argv) {
    if (argc != 2) return 2;
    const std::string dir = argv[1];
    auto load = [&](const char *name) { return npy_load(dir + "/" + name + ".npy"); };
    try {
        const auto m = load("meta").as_vector<int>();  // H nh nkv hd bits page npages batch max_pages n steps window sinks
        const int H = m[0], nh = m[1], nkv = m[2], hd = m[3], bits = m[4], page = m[5], npages = m[6], B = m[7], M = m[8], n = m[9], steps = m[10], window = m[11], sinks = m[12];
        const int qkv = (nh + 2 * nkv) * hd;
        auto block = [&](std::shared_ptr<et::KvCache> cache) {
            auto weight = [&](const char *name, int out, int in) { return w4_mat(out, in, 32, et::DeviceBuffer<half>(as_half(load(name).as_vector<float>()))); };
            auto lq = std::make_unique<Linear<w4_mat>>(H, qkv, weight("wqkv", qkv, H), as_half(load("bqkv").as_vector<float>()).data(), B * n);
            auto lo = std::make_unique<Linear<w4_mat>>(nh * hd, H, weight("wo", H, nh * hd), as_half(load("bo").as_vector<float>()).data(), B * n);
            return std::make_unique<et::CachedAttention<w4_mat, w4_mat>>(std::move(lq), std::move(lo), cache, nh, M, B, n, window, sinks, true);
        };
        auto cache = std::make_shared<et::KvCache>(nkv, hd, bits, page, npages), cache2 = std::make_shared<et::KvCache>(nkv, hd, bits, page, npages);
        auto layer = block(cache), layer2 = block(cache2);
        et::KvPages pages(*cache, B, M);
        et::GuessedTokens tree(B, n);
        et::DeviceBuffer<int> starts(std::vector<int>((std::size_t)B, 0)), counts((std::size_t)B), next((std::size_t)B), next_starts((std::size_t)B);
        et::DeviceBuffer<int> parents((std::size_t)B * n), tokens((std::size_t)B * n), choices((std::size_t)B * n);
        et::DeviceBuffer<half> x((std::size_t)B * n * H), y((std::size_t)B * n * H), out((std::size_t)B * n * H);
        et::KvStep s;
        s.starts = starts.get(), s.counts = counts.get(), s.batch = B, s.n = n, s.window = window, s.sinks = sinks;
        et::stream_t stream = nullptr;
        etChk(et_stream_create(&stream));
        etChk(et_graph_begin_capture(stream));
        pages.give(s, nullptr, nullptr, stream);
        tree.see(s, parents.get(), stream);
        layer->forward(y.get(), x.get(), s, stream);
        layer2->forward(out.get(), y.get(), s, stream);
        tree.follow(s, parents.get(), tokens.get(), choices.get(), next.get(), next_starts.get(), stream);
        tree.keep(s, {cache.get(), cache2.get()}, stream);
        etChk(et_memcpy_d2d(starts.get(), next_starts.get(), starts.bytes(), stream));
        et_graph graph = nullptr;
        etChk(et_graph_end_capture(stream, &graph));
        const auto all_counts = load("counts").as_vector<int>(), all_parents = load("parents").as_vector<int>(), all_tokens = load("tokens").as_vector<int>(),
                   all_choices = load("choices").as_vector<int>();
        const auto all_x = as_half(load("x").as_vector<float>());
        auto put = [&](auto &buffer, const auto &all, int step) { etChk(et_memcpy_h2d(buffer.get(), all.data() + (std::size_t)step * buffer.size, buffer.bytes())); };
        for (int i = 0; i < steps; i++) {
            put(counts, all_counts, i), put(parents, all_parents, i), put(tokens, all_tokens, i), put(choices, all_choices, i), put(x, all_x, i);
            etChk(et_graph_launch(graph, stream));
            etChk(et_stream_sync(stream));
            const auto h = out.to_host();
            std::vector<float> f(h.size());
            for (std::size_t k = 0; k < h.size(); k++) f[k] = static_cast<float>(h[k]);
            npy_save(dir + "/out_" + std::to_string(i) + ".npy", f.data(), "<f4", 4, {(std::size_t)B * n, (std::size_t)H});
            const auto at = starts.to_host(), table = et::DeviceBuffer<int>::from_device(pages.table(), (std::size_t)B * M).to_host();
            npy_save(dir + "/starts_" + std::to_string(i) + ".npy", at.data(), "<i4", 4, {1, (std::size_t)B});
            npy_save(dir + "/table_" + std::to_string(i) + ".npy", table.data(), "<i4", 4, {(std::size_t)B, (std::size_t)M});
            if (pages.missing() != 0 || pages.free_pages() < 0 || pages.free_pages() > npages) {
                std::printf("pages are missing\n");
                return 1;
            }
        }
        etChk(et_graph_destroy(graph));
        etChk(et_stream_destroy(stream));
        et::KvStep other = s;
        other.window = window + 1;
        et::KvStep wide = s;
        wide.n = n + 1;
        const bool refused = refuses([&] { layer->forward(y.get(), x.get(), other); }) && refuses([&] { tree.see(wide, parents.get()); }) &&
                             refuses([&] { tree.follow(s, parents.get(), tokens.get(), choices.get(), next.get(), starts.get()); }) && refuses([&] { tree.keep(s, {}); }) &&
                             refuses([&] { et::GuessedTokens(B, 257); }) && refuses([&] { et::KvPages(*cache, 0, 1); }) && refuses([&] {
                                 et::KvStep more = s;
                                 more.batch = B + 1;
                                 pages.give(more);
                             });
        std::printf(refused ? "ok\n" : "a step of other sizes was taken\n");
        return refused ? 0 : 1;
    } catch (const std::exception &e) {
        std::fprintf(stderr, "%s\n", e.what());
        return 1;
    }
}
