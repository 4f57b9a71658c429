"""The bits of a tree, the path that stands, the cache moved together over it, and block tables, against plain loops: whole numbers and bytes, equal."""
import ctypes as C

import numpy as np
import pytest

from oracle import decode as D
from oracle import sight as S
from tests import harness as Hn
from tests.harness import up
from tests.test_gpu_kv_cache import DeviceCache, tables
from tests.test_gpu_sight import trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 256])
@pytest.mark.parametrize("shape", ["random", "chain", "star", "roots", "wrong"])
def test_bits_of_trees(et, n, shape):
    B = 5
    parents = trees(n, B, n)
    if shape == "chain":
        parents[:] = np.arange(n) - 1
    elif shape == "star":
        parents[:, 1:] = 0
    elif shape == "roots":
        parents[:, ::3] = -1
    elif shape == "wrong":  # itself, later ones, far outside: no parent
        parents[:, ::2] = np.random.default_rng(n).choice([5, n, n + 7, 2 ** 31 - 1, -2 ** 31, -5, 255], parents[:, ::2].shape)
    counts = np.array([n, n - 1, 0, n + 9, -3], np.int32)
    words = S.seen_words(parents, counts, n)
    out = up(et, np.full_like(words, 0xABCD))
    et.tree_seen(up(et, parents), up(et, counts), out, B, n)
    there = np.arange(n) < np.clip(counts, 0, n)[:, None]
    assert np.array_equal(out.numpy(), np.where(there[..., None], words, 0xABCD))
    et.tree_seen(up(et, parents), None, out, B, n)
    assert np.array_equal(out.numpy(), S.seen_words(parents, [n] * B, n))


@pytest.mark.parametrize("n", [1, 2, 31, 64, 65, 130, 256])
@pytest.mark.parametrize("shape", ["random", "chain", "wrong"])
def test_paths(et, n, shape):
    """Few tokens, so that siblings share one and choices often find a child; the lowest of those wins."""
    B = 9
    r = np.random.default_rng(n)
    parents = trees(n, B, n)
    if shape == "chain":
        parents[:] = np.arange(n) - 1
    if shape == "wrong":
        parents[:, 1::2] = r.choice([5, n, 2 ** 31 - 1, -2 ** 31, -1], parents[:, 1::2].shape)
    tokens, choices = (r.integers(0, 2, (B, n)).astype(np.int32) for _ in range(2))
    if shape == "chain":
        tokens[:4], choices[:4] = 7, 7
    counts = np.array([n, n - 1, 0, n + 9, -3] + [n] * 4, np.int32)
    starts = np.array([0, 5, 2 ** 31 - 1 - n, -7, 3, 100, 1, 2, 3], np.int32)
    out = [up(et, np.full((B, n), 77, np.int32))] + [up(et, np.full(B, 77, np.int32)) for _ in range(3)]
    dev = [up(et, a) for a in (parents, tokens, choices, starts, counts)]
    et.tree_follow(*dev, *out, B, n)
    for got, want in zip(out, S.follow(parents, tokens, choices, starts, counts, n)):
        assert np.array_equal(got.numpy(), want)
    # the starts move on where they are, and without starts and counts
    et.tree_follow(*dev, *out[:3], dev[3], B, n)
    assert np.array_equal(dev[3].numpy(), S.follow(parents, tokens, choices, starts, counts, n)[3])
    et.tree_follow(*dev[:3], None, None, *out, B, n)
    for got, want in zip(out, S.follow(parents, tokens, choices, [0] * B, [n] * B, n)):
        assert np.array_equal(got.numpy(), want)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("nkv,hd,page,n,layers", [(1, 32, 16, 1, 1), (12, 64, 16, 16, 1), (3, 96, 48, 7, 3), (2, 256, 32, 64, 2), (5, 160, 16, 130, 1), (2, 128, 64, 256, 1), (1, 64, 16, 5, 70)])
def test_moved_together(et, bits, nkv, hd, page, n, layers):
    """Ascending paths, others, the same place twice, rows and places that are none: the bytes of every layer."""
    r = np.random.default_rng(n)
    B = 6
    starts = np.array([0, 5, 3 * page - 2, -2, 40, 7], np.int32)
    max_pages = -(-(max(starts) + n) // page)
    npages = B * max_pages + 1
    table = tables(1, B, max_pages, npages)
    table[4, -1] = -1
    hosts, devs = [], []
    for layer in range(layers):
        host = D.Cache(bits, nkv, hd, page, npages)
        for a in (host.k_codes, host.v_codes):
            a[:] = r.integers(0, 256, a.shape)
        for a in (host.k_scales, host.v_scales):
            a[:] = r.standard_normal(a.shape)
        hosts.append(host)
        devs.append(DeviceCache(et, host))
    path = np.full((B, n), -1, np.int32)
    kept = np.zeros(B, np.int32)
    for b in range(B):
        way = S.ways(trees(b, 1, n)[0], n)[-1]
        path[b, :len(way)], kept[b] = way, len(way)
    path[1], kept[1] = r.permutation(n), n       # any order: every place comes from another
    path[2], kept[2] = n - 1, n + 5               # all from one place
    if n > 4:
        path[5, :5], kept[5] = [4, -3, n, 2 ** 31 - 1, 0], 5
    et.kv_keep([d.c for d in devs], up(et, table), max_pages, up(et, starts), up(et, path), up(et, kept), B, n)
    for host, dev in zip(hosts, devs):
        S.keep(host, table, starts, path, kept, n)
        dev.same()
    kept[:] = [-1, 0, 1, 0, 0, 0]
    et.kv_keep((et.KvCache * layers)(*(d.c for d in devs)), up(et, table), max_pages, None, up(et, path), up(et, kept), B, n)
    for host, dev in zip(hosts, devs):
        S.keep(host, table, [0] * B, path, kept, n)
        dev.same()


def check_tables(et, before, page, npages, starts, counts, shared, n, window, sinks, ring, state, in_place):
    B, M = before.shape
    want = S.tables(before, page, npages, starts, counts, shared, n, window, sinks, ring, state)
    d_before, d_ring, d_state = up(et, before), up(et, ring), up(et, state)
    d_table = d_before if in_place else up(et, np.full_like(before, 12345))
    d_next = d_state if in_place else up(et, np.full(3, 12345, np.int32))
    slots = up(et, np.full((B, max(n, 1)), 12345, np.int64))
    need = et.kv_tables_workspace(M, B)
    et.kv_tables(d_before, d_table, M, page, npages, up(et, np.array(starts, np.int32)), up(et, np.array(counts, np.int32)), None if shared is None else up(et, np.array(shared, np.int32)),
                 B, n, window, sinks, d_ring, d_state, d_next, slots if n else None, up(et, np.full(max(need, 16), 0xFF, np.uint8)), need)
    got = d_table.numpy(), d_ring.numpy(), d_next.numpy(), slots.numpy()[:, :n]
    for name, g, w in zip(("table", "ring", "state", "slots"), got, want):
        assert np.array_equal(g, w), (name, np.argwhere(g != w)[:5])
    if not in_place:
        assert np.array_equal(d_before.numpy(), before)
    return want


# (sequences, pages of each, tokens of a page, rows): one workgroup, its largest tables and those beyond, more sequences than it takes
SIZES = [(1, 1, 1, 1), (3, 7, 16, 20), (8, 64, 16, 1), (2, 333, 48, 300), (512, 32, 16, 3), (513, 5, 4, 9), (600, 3, 16, 40), (2, 8193, 16, 70), (37, 1000, 64, 500), (1, 70000, 16, 5)]


@pytest.mark.parametrize("B,M,page,n", SIZES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4), (1, 0), (40, 70)])
def test_tables_step_by_step(et, B, M, page, n, window, sinks):
    """Sequences go on, fall back, end and begin; pages run out and come back; every step's table, ring, state and slots."""
    r = np.random.default_rng(B + M)
    npages = max(4, B * M // 2)
    table, ring, state = np.full((B, M), -1, np.int32), r.permutation(npages).astype(np.int32), np.array([npages - 1, npages, 0], np.int32)
    shared = r.integers(0, 3, B) if B > 8 else None
    most = max(1, M * page - n)
    starts = np.zeros(B, np.int64)
    for step in range(6):
        counts = r.integers(0, n + 1, B)
        over = r.random(B) < 0.2
        starts, counts = np.where(over, 0, starts), np.where(over, 0, counts)
        table, ring, state, _ = check_tables(et, table, page, npages, starts, counts, shared, n, window, sinks, ring, state, step % 2 == 1)
        starts = np.where(r.random(B) < 0.3, r.integers(0, most, B), starts + counts - r.integers(0, 2, B))
        starts = np.clip(starts, 0, most)


def test_tables_of_odd_arguments(et):
    """Rows in front of the first position and behind the last page, counts out of range, entries that are no pages, a ring that is none, no rows."""
    r = np.random.default_rng(5)
    before = r.choice([-1, 0, 1, 2, 3, 99, -2 ** 31, 2 ** 31 - 1], (4, 6)).astype(np.int32)
    for s in ([-3, 90, 2 ** 31 - 1, -2 ** 31], [0, 0, 95, 50]):
        for c in ([5, 70, -4, 3], [0, 0, 0, 0]):
            for state in ([7, 5, 0], [-9, 3, 1], [2 ** 31 - 1, 99, 0], [3, -4, 0]):
                for shared in (None, [9, -1, 2, 6]):
                    check_tables(et, before, 16, 8, s, c, shared, 9, 20, 17, np.arange(8, dtype=np.int32), np.array(state, np.int32), False)
    check_tables(et, before, 16, 8, [1, 2, 3, 4], [0] * 4, None, 0, 0, 0, np.arange(8, dtype=np.int32), np.array([1, 4, 0], np.int32), True)
    # a page held twice: given back twice, as far as the ring has room
    check_tables(et, np.zeros((4, 6), np.int32), 16, 8, [0] * 4, [0] * 4, None, 1, 0, 0, np.arange(8, dtype=np.int32), np.array([1, 4, 0], np.int32), True)
    # no sequences: the state is passed on
    check_tables(et, np.zeros((0, 6), np.int32), 16, 8, [], [], None, 1, 0, 0, np.arange(8, dtype=np.int32), np.array([9, 4, 3], np.int32), False)
    # neither starts nor counts: n tokens of each
    d = [up(et, a) for a in (np.full((3, 2), -1, np.int32), np.arange(8, dtype=np.int32), np.array([6, 8, 0], np.int32))]
    et.kv_tables(d[0], d[0], 2, 16, 8, None, None, None, 3, 17, 0, 0, d[1], d[2], d[2])
    assert d[0].numpy().tolist() == [[6, 7], [0, 1], [2, 3]] and d[2].numpy().tolist() == [4, 2, 0]


def test_tables_of_slots_beyond_32_bits(et):
    page, npages = 1 << 20, 1 << 20
    table = np.array([[npages - 1, 3]], np.int32)
    check_tables(et, table, page, npages, [page - 2], [4], None, 4, 0, 0, np.zeros(npages, np.int32), np.array([0, 0, 0], np.int32), False)


def test_tables_in_a_graph(et):
    """A step recorded once and replayed with starts moving on: every replay as eager calls on a second set; one launch, and two."""
    lib = et.lib()
    for B, M in ((5, 40), (5, 5000)):
        page, n, npages = 16, 9, 5 * 60
        stream = C.c_void_p()
        et.check(lib.et_stream_create(C.byref(stream)))
        need = et.kv_tables_workspace(M, B)
        sets = [[up(et, a) for a in (np.full((B, M), -1, np.int32), np.arange(npages, dtype=np.int32), np.array([0, npages, 0], np.int32), np.zeros((B, n), np.int64), np.zeros(max(16, need), np.uint8))]
                for _ in range(2)]
        starts, counts = up(et, np.zeros(B, np.int32)), up(et, np.zeros(B, np.int32))

        def step(s, at):
            et.kv_tables(s[0], s[0], M, page, npages, starts, counts, None, B, n, 60, 20, s[1], s[2], s[2], s[3], s[4], need, at)

        et.check(lib.et_graph_begin_capture(stream))
        step(sets[0], stream)
        graph = C.c_void_p()
        et.check(lib.et_graph_end_capture(stream, C.byref(graph)))
        at = np.zeros(B, np.int32)
        r = np.random.default_rng(2)
        for rep in range(8):
            now = r.integers(0, n + 1, B).astype(np.int32)
            for buf, a in ((starts, at), (counts, now)):
                et.check(lib.et_memcpy_h2d(buf.ptr, a.ctypes.data, a.nbytes))
            et.check(lib.et_graph_launch(graph, stream))
            step(sets[1], stream)
            et.check(lib.et_stream_sync(stream))
            for a, b in zip(*sets):
                assert np.array_equal(a.numpy(), b.numpy())
            at = (at + now).astype(np.int32)
        et.check(lib.et_graph_destroy(graph))
        et.check(lib.et_stream_destroy(stream))
