"""Guessing several tokens at once, as a server does it: pages handed out, a tree's keys and values written, attention of its nodes, the path that stands, what stands moved
together, and on from there, all of it on the device.  Eager calls, a graph of the same calls and the class layer give the same bits, and what stands is what the layer gives on
the whole sequence in binary64."""
import ctypes as C
import subprocess

import numpy as np
import pytest

from oracle import decode as D
from oracle import sight as S
from tests import harness as Hn
from tests.harness import up
from tests.test_gpu_decode import EXE, Device, Layer

pytestmark = pytest.mark.gpu


def attention_block(layer, bits, x, window, sinks):
    """The attention block (projection, attention, output projection) on one sequence, in binary64."""
    lin = lambda k, x: x @ layer.value[k].T + layer.bias[k].astype(np.float64)  # noqa: E731
    nh, nkv, hd = layer.nh, layer.nkv, layer.hd
    qkv = lin("qkv", x.astype(np.float64))
    kept = lambda a: D.stands_for(*D.quantise(a.astype(np.float16).reshape(-1, nkv, hd), 2 ** bits - 1))  # noqa: E731
    q, k, v = qkv[:, :nh * hd].reshape(-1, nh, hd), kept(qkv[:, nh * hd:(nh + nkv) * hd]), kept(qkv[:, (nh + nkv) * hd:])
    z = np.zeros((len(x), nh, hd))
    at = np.arange(len(x))
    for i in range(len(x)):
        seen = (at <= i) & ((at > i - window) | (at < sinks) if window else True)
        for h in range(nh):
            s = np.where(seen, k[:, h * nkv // nh] @ q[i, h] / np.sqrt(hd), -np.inf)
            p = np.exp(s - s.max())
            z[i, h] = (p / p.sum()) @ v[:, h * nkv // nh]
    return lin("o", z.reshape(len(x), -1))


class Server:
    """Buffers of a batch of sequences, and a step over them."""

    def __init__(self, et, layer, bits, page, npages, B, max_pages, n, window, sinks):
        self.et, self.L, self.sizes = et, layer, (B, max_pages, n, window, sinks)
        self.dev = Device(et, layer, bits, page, B, max_pages, seed=1)
        self.host = D.Cache(bits, layer.nkv, layer.hd, page, npages, fill=0xFF)
        self.bufs = [up(et, getattr(self.host, k)) for k in ("k_codes", "k_scales", "v_codes", "v_scales")]
        self.cache = et.KvCache(*(b.ptr for b in self.bufs), bits, layer.nkv, layer.hd, page, npages)
        self.page, self.npages = page, npages
        i32 = lambda *s: up(et, np.full(s, -1, np.int32))  # noqa: E731
        self.table, self.ring, self.state = i32(B, max_pages), up(et, np.arange(npages, dtype=np.int32)), up(et, np.array([0, npages, 0], np.int32))
        self.starts, self.counts, self.next_starts, self.kept, self.next = (up(et, np.zeros(B, np.int32)) for _ in range(5))
        self.parents, self.tokens, self.choices, self.path = (i32(B, n) for _ in range(4))
        self.slots, self.seen = up(et, np.zeros((B, n), np.int64)), up(et, np.zeros((B, n, (n + 31) // 32), np.uint32))
        self.x, self.qkv, self.z, self.y = (up(et, np.zeros((B * n, w), np.float16)) for w in (layer.H, layer.qkv, layer.nh * layer.hd, layer.H))
        self.need = et.mha_kv_tree_workspace(self.cache, max_pages, B, n, layer.nh, window, sinks)
        self.tables_need = et.kv_tables_workspace(max_pages, B)
        self.ws, self.tables_ws = up(et, np.full(max(16, self.need), 0xFF, np.uint8)), up(et, np.zeros(max(16, self.tables_need), np.uint8))

    def linear(self, k, x, y, stream):
        codes, scales, bias = self.dev.w[k]
        out, n_in = self.L.shape[k]
        self.et.linear_w4(codes, scales, self.L.group, bias, x, y, None, self.sizes[0] * self.sizes[2], n_in, out, 0, stream)

    def step(self, stream=None):
        et, L, (B, M, n, window, sinks) = self.et, self.L, self.sizes
        et.kv_tables(self.table, self.table, M, self.page, self.npages, self.starts, self.counts, None, B, n, window, sinks, self.ring, self.state, self.state, self.slots, self.tables_ws,
                     self.tables_need, stream)
        et.tree_seen(self.parents, self.counts, self.seen, B, n, stream)
        self.linear("qkv", self.x, self.qkv, stream)
        where = (self.cache, self.table, M, self.starts, self.counts)
        et.kv_write(*where, self.qkv.offset(2 * L.nh * L.hd), self.qkv.offset(2 * (L.nh + L.nkv) * L.hd), L.qkv, L.qkv, B, n, stream)
        et.mha_kv_tree(*where, self.seen, self.qkv, L.qkv, self.z, L.nh * L.hd, B, n, L.nh, window, sinks, L.hd ** -0.5, self.ws, self.need, stream)
        self.linear("o", self.z, self.y, stream)
        et.tree_follow(self.parents, self.tokens, self.choices, self.starts, self.counts, self.path, self.kept, self.next, self.next_starts, B, n, stream)
        et.kv_keep([self.cache], self.table, M, self.starts, self.path, self.kept, B, n, stream)
        et.check(et.lib().et_memcpy_d2d(self.starts.ptr, self.next_starts.ptr, 4 * B, stream))

    def put(self, **arrays):
        for k, a in arrays.items():
            a = np.ascontiguousarray(a)
            self.et.check(self.et.lib().et_memcpy_h2d(getattr(self, k).ptr, a.ctypes.data, a.nbytes))

    def results(self):
        return {k: getattr(self, k).numpy() for k in ("table", "ring", "state", "slots", "path", "kept", "next", "starts", "seen")}


class Plan:
    """Trees whose nodes' tokens are partly what a sequence goes on with, and what the model chose after each node."""

    def __init__(self, B, n, vocabulary, seed):
        self.B, self.n, self.V, self.r = B, n, vocabulary, np.random.default_rng(seed)
        self.said = [[] for _ in range(B)]  # of each sequence: the tokens that stand
        self.next = self.r.integers(0, vocabulary, B)

    def step(self, counts):
        r, n = self.r, self.n
        parents, tokens, choices = np.full((self.B, n), -1, np.int32), r.integers(0, self.V, (self.B, n)).astype(np.int32), r.integers(0, self.V, (self.B, n)).astype(np.int32)
        for b in range(self.B):
            tokens[b, 0] = self.next[b]
            for i in range(1, n):
                parents[b, i] = max(0, i - 1 - int(r.integers(0, 3)))
                if r.random() < 0.7 and i < counts[b]:
                    tokens[b, i] = choices[b, parents[b, i]]
        return parents, tokens, choices


# (bits, page, key/value heads' queries, nodes, window, first tokens): kernels for few rows, several and many
CASES = [(4, 16, 2, 6, 0, 0), (8, 32, 4, 9, 40, 5), (4, 16, 2, 40, 0, 0), (4, 48, 4, 40, 64, 3), (8, 16, 4, 33, 33, 0)]


@pytest.mark.parametrize("bits,page,per,n,window,sinks", CASES)
def test_guessing_on_the_device(et, bits, page, per, n, window, sinks):
    """Eight steps of three sequences; the second ends after the fourth step and another begins in its place."""
    lib, nkv, hd, B, M, V = et.lib(), 2, 64, 3, 24, 40
    layer = Layer(256, nkv * per, nkv, hd, 64, 64, seed=bits + n)
    npages = B * 12
    eager, replayed = (Server(et, layer, bits, page, npages, B, M, n, window, sinks) for _ in range(2))
    words = Hn.randn((V, layer.H), 9)
    plan = Plan(B, n, V, seed=n)
    stream = C.c_void_p()
    et.check(lib.et_stream_create(C.byref(stream)))
    et.check(lib.et_graph_begin_capture(stream))
    replayed.step(stream)
    graph = C.c_void_p()
    et.check(lib.et_graph_end_capture(stream, C.byref(graph)))
    starts, worst = np.zeros(B, np.int32), 0.0
    held = (np.full((B, M), -1, np.int32), np.arange(npages, dtype=np.int32), np.array([0, npages, 0], np.int32))
    for step in range(8):
        counts = np.array([n, max(1, n - step), n // 2 + 1], np.int32)
        if step == 4:
            starts[1] = counts[1] = 0
            plan.said[1] = []
        parents, tokens, choices = plan.step(counts)
        x = words[tokens.ravel()]
        for s in (eager, replayed):
            s.put(starts=starts, counts=counts, parents=parents, tokens=tokens, choices=choices, x=x)
        eager.step()
        et.check(lib.et_graph_launch(graph, stream))
        et.check(lib.et_stream_sync(stream))
        et.check(lib.et_device_sync())
        got = eager.results()
        for k, a in replayed.results().items():
            assert np.array_equal(a, got[k]), (step, k)
        y = eager.y.numpy().reshape(B, n, -1)
        assert np.array_equal(y.view(np.uint16), replayed.y.numpy().reshape(B, n, -1).view(np.uint16)), step
        # tables, path and positions as the oracle has them
        table, ring, state, slots = S.tables(held[0], page, npages, starts, counts, None, n, window, sinks, *held[1:])
        held = (table, ring, state)
        assert state[2] == 0 and np.array_equal(got["table"], table) and np.array_equal(got["state"], state) and np.array_equal(got["slots"], slots)
        free = [got["ring"][(state[0] + i) % npages] for i in range(state[1])]
        assert free == [ring[(state[0] + i) % npages] for i in range(state[1])] and sorted(free + [p for p in table.ravel() if p >= 0]) == list(range(npages))
        path, kept, token, on = S.follow(parents, tokens, choices, starts, counts, n)
        assert np.array_equal(got["path"], path) and np.array_equal(got["kept"], kept) and np.array_equal(got["next"], token) and np.array_equal(got["starts"], on)
        # the nodes that stand, and two that do not, against the block on the sequence that leads to them
        for b in range(B):
            if counts[b] == 0:
                continue
            wanted = list(path[b, :kept[b]][-1:]) + list(plan.r.integers(0, counts[b], 2))
            for node in wanted:
                way = [node]
                while way[-1] > 0:
                    way.append(parents[b, way[-1]])
                way = way[::-1]
                sequence = plan.said[b] + [tokens[b, i] for i in way]
                want = attention_block(layer, bits, words[sequence], window, sinks)[-len(way):]
                worst = max(worst, Hn.max_abs(y[b, way], want))
            plan.said[b] += [tokens[b, i] for i in path[b, :kept[b]]]
            plan.next[b] = token[b]
        starts = on
    assert max(len(s) for s in plan.said) > 12
    # what a cache rounds and what a projection of 256 or so binary16 numbers rounds: the 2e-2 that a layer is held to
    assert worst <= 2e-2, worst
    et.check(lib.et_graph_destroy(graph))
    et.check(lib.et_stream_destroy(stream))


def test_class_layer_guesses(et, tmp_path):
    """KvPages, CachedAttention and GuessedTokens of two layers, a step recorded in a graph and replayed: bit for bit what the calls of the C ABI give."""
    exe = EXE.with_name("guess_cases")
    assert exe.exists(), f"{exe} is missing: build it with `python scpaper-2021_amd/build.py`"
    B, n, window, sinks, steps, page, npages, M, V = 3, 8, 24, 4, 6, 16, 18, 12, 30
    layer = Layer(128, 4, 2, 32, 64, 32, seed=4)
    plan, words = Plan(B, n, V, seed=8), Hn.randn((V, layer.H), 9)
    first, second = (Server(et, layer, 4, page, npages, B, M, n, window, sinks) for _ in range(2))
    f32 = lambda a: np.asarray(a, np.float32)  # noqa: E731
    np.save(tmp_path / "meta.npy", np.array([layer.H, layer.nh, layer.nkv, layer.hd, 4, page, npages, B, M, n, steps, window, sinks], np.int32))
    for name, a in (("wqkv", layer.dense["qkv"]), ("wo", layer.dense["o"]), ("bqkv", layer.bias["qkv"]), ("bo", layer.bias["o"])):
        np.save(tmp_path / f"{name}.npy", f32(a))
    want, inputs = [], []
    for step in range(steps):
        counts = np.array([n, n - step, step + 1], np.int32)
        parents, tokens, choices = plan.step(counts)
        x = words[tokens.ravel()]
        inputs.append((counts, parents, tokens, choices, x))
        for s, rows in ((first, x), (second, None)):
            s.put(counts=counts, parents=parents, tokens=tokens, choices=choices, x=first.y.numpy() if rows is None else rows)
            s.step()
            et.check(et.lib().et_device_sync())
        got = second.results()
        plan.next = got["next"].astype(np.int64)
        want.append((second.y.numpy(), got))
    for i, name in enumerate(("counts", "parents", "tokens", "choices")):
        np.save(tmp_path / f"{name}.npy", np.stack([a[i].reshape(-1) for a in inputs]).astype(np.int32))
    np.save(tmp_path / "x.npy", f32(np.stack([a[4] for a in inputs]).reshape(steps, -1)))
    res = subprocess.run([str(exe), str(tmp_path)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and "ok" in res.stdout, res.stdout + res.stderr
    for i, (y, got) in enumerate(want):
        valid = np.arange(n)[None] < inputs[i][0][:, None]
        assert np.array_equal(np.load(tmp_path / f"out_{i}.npy").reshape(B, n, -1)[valid], f32(y).reshape(B, n, -1)[valid]), i
        assert np.array_equal(np.load(tmp_path / f"starts_{i}.npy").ravel(), got["starts"]) and np.array_equal(np.load(tmp_path / f"table_{i}.npy").reshape(B, M), got["table"]), i
