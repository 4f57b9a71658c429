"""Generating token by token: the cache, the attention over it and 4-bit Linears run together, as a decoder layer's step through the C ABI and
as the class layer's CachedAttention."""
import subprocess
from pathlib import Path

import numpy as np
import pytest

from oracle import decode as D
from tests import harness as Hn
from tests.harness import up

pytestmark = pytest.mark.gpu

EXE = Path(__file__).resolve().parent / "cpp" / "bin" / "decode_cases"


class Layer:
    """A causal decoder layer with 4-bit weights: attention, SkipLayerNorm, GELU feed-forward, SkipLayerNorm."""

    def __init__(self, H, nh, nkv, hd, FF, group, seed):
        r = np.random.default_rng(seed)
        w = lambda out, n_in: (r.standard_normal((out, n_in)) * n_in ** -0.5).astype(np.float16)  # noqa: E731
        self.H, self.nh, self.nkv, self.hd, self.FF, self.group = H, nh, nkv, hd, FF, group
        self.qkv = (nh + 2 * nkv) * hd
        self.shape = {"qkv": (self.qkv, H), "o": (H, nh * hd), "up": (FF, H), "down": (H, FF)}
        self.dense = {k: w(*s) for k, s in self.shape.items()}
        self.bias = {k: (r.standard_normal(s[0]) * 0.1).astype(np.float16) for k, s in self.shape.items()}
        self.norm = [((1 + 0.1 * r.standard_normal(H)).astype(np.float16), (0.1 * r.standard_normal(H)).astype(np.float16)) for _ in range(2)]
        self.packed = {k: D.w4_pack(v, group) for k, v in self.dense.items()}
        self.value = {k: D.w4_dense(*v, group) for k, v in self.packed.items()}


class Device:
    """A layer and a cache of it on the device."""

    def __init__(self, et, layer, bits, page, B, max_pages, seed):
        self.et, self.L, self.B, self.max_pages = et, layer, B, max_pages
        self.npages = B * max_pages + 1
        self.table = np.random.default_rng(seed).permutation(self.npages)[:B * max_pages].reshape(B, max_pages).astype(np.int32)
        self.host = D.Cache(bits, layer.nkv, layer.hd, page, self.npages)
        self.bufs = [up(et, getattr(self.host, k)) for k in ("k_codes", "k_scales", "v_codes", "v_scales")]
        self.cache = et.KvCache(*(b.ptr for b in self.bufs), bits, layer.nkv, layer.hd, page, self.npages)
        self.w = {}
        for k, (out, n_in) in layer.shape.items():
            dense, codes, scales = up(et, layer.dense[k]), up(et, np.zeros((out, n_in // 2), np.uint8)), up(et, np.zeros((n_in // layer.group, out, 2), np.float16))
            et.dense_to_w4(dense, codes, scales, n_in, out, layer.group)
            self.w[k] = (codes, scales, up(et, layer.bias[k]))
        self.norm = [tuple(up(et, a) for a in g) for g in layer.norm]
        self.d_table = up(et, self.table)

    def linear(self, k, x, T, act=0):
        et, (out, n_in) = self.et, self.L.shape[k]
        y = up(et, np.zeros((T, out), np.float16))
        codes, scales, bias = self.w[k]
        et.linear_w4(codes, scales, self.L.group, bias, x, y, None, T, n_in, out, act)
        return y

    def attention(self, x, starts, counts, n):
        """The attention block: what CachedAttention runs."""
        et, L, T = self.et, self.L, self.B * n
        qkv = self.linear("qkv", x, T)
        where = (self.cache, self.d_table, self.max_pages, None if starts is None else up(et, np.array(starts, np.int32)),
                 None if counts is None else up(et, np.array(counts, np.int32)))
        et.kv_write(*where, qkv.offset(2 * L.nh * L.hd), qkv.offset(2 * (L.nh + L.nkv) * L.hd), L.qkv, L.qkv, self.B, n)
        z = up(et, np.zeros((T, L.nh * L.hd), np.float16))
        need = et.mha_kv_workspace(self.cache, self.max_pages, self.B, n, L.nh)
        et.mha_kv(*where, qkv, L.qkv, z, L.nh * L.hd, self.B, n, L.nh, L.hd ** -0.5, et.MHA_CAUSAL, up(et, np.zeros(max(16, need), np.uint8)), need)
        return self.linear("o", z, T)

    def step(self, x, starts, counts, n):
        et, L, T = self.et, self.L, self.B * n
        dx = up(et, x)
        a, h = self.attention(dx, starts, counts, n), up(et, np.zeros((T, L.H), np.float16))
        et.skip_layernorm(h, a, dx, *self.norm[0], T, L.H)
        f = self.linear("down", self.linear("up", h, T, act=et.ACT_GELU), T)
        out = up(et, np.zeros((T, L.H), np.float16))
        et.skip_layernorm(out, f, h, *self.norm[1], T, L.H)
        return out.numpy()


def norm(x, g, b):
    x = x - x.mean(-1, keepdims=True)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * g.astype(np.float64) + b.astype(np.float64)


def reference(layer, bits, tokens):
    """The layer on one sequence's tokens in binary64, with the weights that the codes stand for and keys and values through the cache's format."""
    lin = lambda k, x: x @ layer.value[k].T + layer.bias[k].astype(np.float64)  # noqa: E731
    nh, nkv, hd = layer.nh, layer.nkv, layer.hd
    x = tokens.astype(np.float64)
    qkv = lin("qkv", x)
    kept = lambda a: D.stands_for(*D.quantise(a.astype(np.float16).reshape(-1, nkv, hd), 2 ** bits - 1))  # noqa: E731
    q, k, v = qkv[:, :nh * hd].reshape(-1, nh, hd), kept(qkv[:, nh * hd:(nh + nkv) * hd]), kept(qkv[:, (nh + nkv) * hd:])
    z = np.zeros((len(x), nh, hd))
    for i in range(len(x)):
        for h in range(nh):
            g = h * nkv // nh
            s = k[:i + 1, g] @ q[i, h] / np.sqrt(hd)
            p = np.exp(s - s.max())
            z[i, h] = (p / p.sum()) @ v[:i + 1, g]
    h = norm(lin("o", z.reshape(len(x), -1)) + x, *layer.norm[0])
    u = lin("up", h)
    u = u * (0.5 + 0.5 * np.tanh(u * (0.035677408136 * u * u + 0.7978845608028654)))
    return norm(lin("down", u) + h, *layer.norm[1])


@pytest.mark.parametrize("bits,page,group", [(4, 16, 64), (8, 48, 32), (4, 64, 128)])
def test_decoder_layer_token_by_token(et, bits, page, group):
    """Prompts of unequal length in pieces, then single tokens, against the layer on whole sequences in binary64, to the 2e-2 that a layer in binary16 is
    held to."""
    layer = Layer(256, 8, 4, 64, 512, group, seed=bits + page)
    B, lengths = 3, [37, 20, 29]
    total = [l + 6 for l in lengths]
    seqs = [Hn.randn((t, layer.H), 40 + b) for b, t in enumerate(total)]
    dev = Device(et, layer, bits, page, B, -(-max(total) // page), seed=1)
    want = [reference(layer, bits, s) for s in seqs]
    worst = 0.0
    done = [0] * B
    n = 13
    while any(d < l for d, l in zip(done, lengths)):  # pieces of 13 rows, the last ones short, some empty
        counts = [min(n, l - d) for d, l in zip(done, lengths)]
        x = np.full((B, n, layer.H), np.nan, np.float16)
        for b in range(B):
            x[b, :counts[b]] = seqs[b][done[b]:done[b] + counts[b]]
            x[b, counts[b]:] = 0
        got = dev.step(x.reshape(B * n, -1), done, counts, n).reshape(B, n, -1)
        for b in range(B):
            worst = max(worst, Hn.max_abs(got[b, :counts[b]], want[b][done[b]:done[b] + counts[b]]))
            done[b] += counts[b]
    for i in range(6):
        got = dev.step(np.stack([seqs[b][lengths[b] + i] for b in range(B)]), [l + i for l in lengths], None, 1)
        for b in range(B):
            worst = max(worst, Hn.max_abs(got[b], want[b][lengths[b] + i]))
    assert worst <= 2e-2, worst


def test_class_layer_runs_the_same_calls(et, tmp_path):
    """CachedAttention with 4-bit projections, its steps recorded in a graph: bit for bit what the calls of the C ABI give."""
    H, nh, nkv, hd, bits, page, B, max_pages, prompt, steps = 128, 4, 2, 32, 4, 16, 2, 3, 9, 4
    layer = Layer(H, nh, nkv, hd, 64, 32, seed=3)
    dev = Device(et, layer, bits, page, B, max_pages, seed=5)
    counts = [9, 5]
    x, tokens = Hn.randn((B * prompt, H), 6), Hn.randn((steps, B, H), 7)
    f32 = lambda a: np.asarray(a, np.float32)  # noqa: E731
    np.save(tmp_path / "meta.npy", np.array([H, nh, nkv, hd, bits, page, dev.npages, B, max_pages, prompt, steps], np.int32))
    np.save(tmp_path / "table.npy", dev.table)
    np.save(tmp_path / "counts.npy", np.array(counts, np.int32))
    for name, a in (("wqkv", layer.dense["qkv"]), ("wo", layer.dense["o"]), ("bqkv", layer.bias["qkv"]), ("bo", layer.bias["o"]), ("prompt", x), ("tokens", tokens)):
        np.save(tmp_path / f"{name}.npy", f32(a))
    assert EXE.exists(), f"{EXE} is missing: build it with `python scpaper-2021_amd/build.py`"
    res = subprocess.run([str(EXE), str(tmp_path)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and "ok" in res.stdout, res.stdout + res.stderr
    want = dev.attention(up(et, x), None, counts, prompt).numpy().reshape(B, prompt, H)
    got = np.load(tmp_path / "out_prompt.npy").reshape(B, prompt, H)
    for b in range(B):
        assert np.array_equal(got[b, :counts[b]], f32(want[b, :counts[b]]))
    for i in range(steps):
        want = dev.attention(up(et, tokens[i]), [c + i for c in counts], None, 1).numpy()
        assert np.array_equal(np.load(tmp_path / f"out_{i}.npy"), f32(want)), i


def test_class_layer_sizes():
    """CachedAttention with tile-sparse projections, with fewer pages than it was made for, and what it refuses when it is made."""
    exe = EXE.with_name("cached_attention_sizes")
    assert exe.exists(), f"{exe} is missing: build it with `python scpaper-2021_amd/build.py`"
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and "ok" in res.stdout, res.stdout + res.stderr
