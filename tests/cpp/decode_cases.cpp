// Generating token by token through the C++ class layer: a CachedAttention block with 4-bit
// projections over a paged cache, driven as a server drives it (a piece of every prompt, then
// single tokens), and the results written as .npy files for the Python side to compare.
// Usage: decode_cases <dir>
#include <cstdio>
#include <string>

#include "et/Cached_attention.h"
#include "et/npy.hpp"

using et::npy::npy_load;
using et::npy::npy_save;

static std::vector<half> load_half(const std::string &path) {
    const auto f = npy_load(path).as_vector<float>();
    std::vector<half> h(f.size());
    for (std::size_t i = 0; i < f.size(); i++) h[i] = static_cast<half>(f[i]);
    return h;
}
static std::vector<int> load_int(const std::string &path) { return npy_load(path).as_vector<int>(); }

template <typename W> static std::unique_ptr<et::CachedAttention<W, W>> block(const std::string &dir, std::shared_ptr<et::KvCache> cache, int H, int nh, int nkv, int hd,
                                                                              int max_pages, int batch, int n) {
    const int qkv = (nh + 2 * nkv) * hd;
    auto weight = [&](const char *name, int out, int in) { return w4_mat(out, in, 32, et::DeviceBuffer<half>(load_half(dir + "/" + name))); };
    auto bias = [&](const char *name) { return load_half(dir + "/" + name); };
    auto lq = std::make_unique<Linear<W>>(H, qkv, weight("wqkv.npy", qkv, H), bias("bqkv.npy").data(), batch * n);
    auto lo = std::make_unique<Linear<W>>(nh * hd, H, weight("wo.npy", H, nh * hd), bias("bo.npy").data(), batch * n);
    return std::make_unique<et::CachedAttention<W, W>>(std::move(lq), std::move(lo), cache, nh, max_pages, batch, n);
}

int main(int argc, char **argv) {
    if (argc != 2) return 2;
    const std::string dir = argv[1];
    try {
        const auto m = load_int(dir + "/meta.npy");  // H nh nkv hd bits page npages batch max_pages prompt steps
        const int H = m[0], nh = m[1], nkv = m[2], hd = m[3], bits = m[4], page = m[5], npages = m[6], B = m[7], max_pages = m[8], prompt = m[9], steps = m[10];
        auto cache = std::make_shared<et::KvCache>(nkv, hd, bits, page, npages);
        const et::DeviceBuffer<int> table(load_int(dir + "/table.npy")), counts(load_int(dir + "/counts.npy"));
        const et::DeviceBuffer<half> x(load_half(dir + "/prompt.npy"));  // [B * prompt x H]
        et::DeviceBuffer<half> y((std::size_t)B * prompt * H);
        auto first = block<w4_mat>(dir, cache, H, nh, nkv, hd, max_pages, B, prompt);
        et::KvStep s;
        s.table = table.get(), s.max_pages = max_pages, s.counts = counts.get(), s.batch = B, s.n = prompt;
        first->forward(y.get(), x.get(), s);
        auto save = [&](const std::string &name, const et::DeviceBuffer<half> &b, std::size_t cols) {
            const auto h = b.to_host();
            std::vector<float> f(h.size());
            for (std::size_t i = 0; i < h.size(); i++) f[i] = static_cast<float>(h[i]);
            npy_save(dir + "/" + name, f.data(), "<f4", 4, {h.size() / cols, cols});
        };
        save("out_prompt.npy", y, (std::size_t)H);
        // single tokens: the step is recorded once, and replayed with the positions moved on
        auto next = block<w4_mat>(dir, cache, H, nh, nkv, hd, max_pages, B, 1);
        const auto tokens = load_half(dir + "/tokens.npy");  // [steps][B x H]
        std::vector<int> at = counts.to_host();
        et::DeviceBuffer<int> starts(at);
        et::DeviceBuffer<half> in((std::size_t)B * H), out((std::size_t)B * H);
        s.starts = starts.get(), s.counts = nullptr, s.n = 1;
        et::stream_t stream = nullptr;
        etChk(et_stream_create(&stream));
        etChk(et_graph_begin_capture(stream));
        next->forward(out.get(), in.get(), s, stream);
        et_graph graph = nullptr;
        etChk(et_graph_end_capture(stream, &graph));
        for (int i = 0; i < steps; i++) {
            etChk(et_memcpy_h2d(in.get(), tokens.data() + (std::size_t)i * B * H, in.bytes()));
            etChk(et_memcpy_h2d(starts.get(), at.data(), starts.bytes()));
            etChk(et_graph_launch(graph, stream));
            etChk(et_stream_sync(stream));
            save("out_" + std::to_string(i) + ".npy", out, (std::size_t)H);
            for (int &a : at) a++;
        }
        etChk(et_graph_destroy(graph));
        etChk(et_stream_destroy(stream));
        bool refused = false;
        try {
            next->forward(out.get(), in.get(), et::KvStep{}, nullptr);
        } catch (const et::Error &) {
            refused = true;
        }
        std::printf(refused ? "ok\n" : "a step of other sizes was taken\n");
        return refused ? 0 : 1;
    } catch (const std::exception &e) {
        std::fprintf(stderr, "%s\n", e.what());
        return 1;
    }
}
