"""What the calls of windows, trees and block tables refuse, before anything is launched; workspaces; and the oracle's own bounds."""
import ctypes as C

import numpy as np
import pytest

from oracle import sight as S
from tests.test_decode_arguments import BAD_CACHE, P, cache


def calls(et, c, table=P, max_pages=4, B=1, n=1, ldq=256, Q=P, Z=P, nh=4, window=32, sinks=4, flags=0, scale=0.1, seen=P, ws=P, ws_bytes=1 << 30):
    lib, ref = et.lib(), C.byref(c)
    return {"window": lib.et_mha_kv_window_f16(ref, table, max_pages, None, None, Q, ldq, Z, ldq, B, n, nh, window, sinks, scale, flags, ws, ws_bytes, None),
            "tree": lib.et_mha_kv_tree_f16(ref, table, max_pages, None, None, seen, Q, ldq, Z, ldq, B, n, nh, window, sinks, scale, ws, ws_bytes, None)}


@pytest.mark.parametrize("bad,status", BAD_CACHE)
def test_caches_that_are_none(et, bad, status):
    c = cache(et, **bad)
    assert set(calls(et, c, ldq=1 << 30, nh=max(1, c.nkv)).values()) == {status}
    size = C.c_size_t()
    for call in (et.lib().et_mha_kv_window_workspace, et.lib().et_mha_kv_tree_workspace):
        assert call(C.byref(c), 4, 1, 1, max(1, c.nkv), 32, 4, C.byref(size)) == status
    assert et.lib().et_kv_keep(C.byref(c), 1, P, 4, None, P, P, 1, 1, None) == status
    assert et.lib().et_last_error().startswith(b"et_kv_keep:")


def test_other_arguments_of_attention(et):
    c = cache(et)
    for bad, status in ((dict(table=None), -1), (dict(table=P + 2), -2), (dict(max_pages=0), -1), (dict(max_pages=1 << 28), -2), (dict(B=-1), -1), (dict(n=-1), -1), (dict(ldq=248), -1),
                        (dict(ldq=260), -2), (dict(Q=P + 8), -2), (dict(Z=P + 8), -2), (dict(Q=None), -1), (dict(Z=None), -1), (dict(nh=3), -1), (dict(nh=0), -1), (dict(sinks=-1), -1),
                        (dict(window=-1), -1), (dict(scale=float("nan")), -1), (dict(scale=2e15), -1), (dict(B=1 << 20), -2)):
        assert set(calls(et, c, **bad).values()) == {status}, bad
    assert calls(et, c, window=0, n=0) == {"window": -1, "tree": 0}
    assert calls(et, c, window=4, n=5, B=0) == {"window": 0, "tree": -1}  # a tree's node must not lose sight of another
    assert calls(et, c, n=257, window=300, B=0) == {"window": 0, "tree": -2} and calls(et, c, n=256, window=0, B=0)["tree"] == 0
    assert calls(et, c, flags=2, n=0)["window"] == -1 and calls(et, c, flags=et.MHA_CAUSAL, n=0)["window"] == 0
    assert calls(et, c, seen=None, n=0)["tree"] == -1 and calls(et, c, seen=P + 1, n=0)["tree"] == -2
    assert set(calls(et, c, B=0).values()) == {0} and set(calls(et, c, n=0).values()) == {0}
    assert set(calls(et, c, B=0, window=0x7fffffff, sinks=0x7fffffff).values()) == {0}


@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4), (4096, 16), (100000, 100000)])
def test_workspaces(et, window, sinks):
    """They do not grow with fewer pages, and a call without one is refused."""
    ask = et.mha_kv_tree_workspace if window == 0 else et.mha_kv_window_workspace
    for nkv, hd, bits, B, n, nh in ((1, 64, 4, 1, 1, 1), (8, 128, 4, 1, 1, 32), (8, 96, 8, 3, 7, 8), (16, 64, 4, 40, 1, 16), (2, 256, 8, 2, 40, 16), (8, 128, 4, 2, 64, 32), (8, 128, 8, 33, 7, 8)):
        c = cache(et, nkv=nkv, hd=hd, bits=bits, npages=1 << 14)
        need = [ask(c, pages, B, n, nh, window, sinks) for pages in [*range(1, 200), *range(200, 9000, 37)]]
        assert need == sorted(need)
    c = cache(et, nkv=1, npages=1 << 16)
    pages = 1 << 16
    need = et.mha_kv_tree_workspace(c, pages, 1, 1, 1)
    assert need > 0
    for ws, have in ((None, need), (P, need - 1), (P + 8, need)):
        assert calls(et, c, max_pages=pages, nh=1, window=0, ws=ws, ws_bytes=have)["tree"] == (-2 if ws == P + 8 else -1), (ws, have)
        assert b"workspace" in et.lib().et_last_error()


def test_trees_and_paths(et):
    lib = et.lib()
    seen = lambda parents=P, seen=P, B=1, n=4: lib.et_tree_seen(parents, None, seen, B, n, None)  # noqa: E731
    for bad, status in ((dict(parents=None), -1), (dict(seen=None), -1), (dict(B=-1), -1), (dict(n=-1), -1), (dict(n=257), -2), (dict(B=65536), -2), (dict(seen=P + 2), -2)):
        assert seen(**bad) == status, bad
    assert seen(B=0) == seen(n=0) == 0
    args = ["parents", "tokens", "choices", "path", "kept", "next_tokens", "next_starts"]

    def follow(B=0, n=4, **bad):
        a = {k: P for k in args} | bad
        return lib.et_tree_follow(a["parents"], a["tokens"], a["choices"], None, None, a["path"], a["kept"], a["next_tokens"], a["next_starts"], B, n, None)

    for k in args:
        assert follow(**{k: None}) == -1
    assert follow(B=-1) == -1 and follow(n=0) == -1 and follow(n=257) == -2 and follow() == 0
    one, other = cache(et), cache(et, bits=8)
    two = (et.KvCache * 2)(one, other)
    assert lib.et_kv_keep(two, 2, P, 4, None, P, P, 1, 4, None) == -1 and b"cache 1" in lib.et_last_error()
    two = (et.KvCache * 2)(one, one)
    for args, status in (((two, 0, P, 4, None, P, P, 1, 4), -1), ((None, 1, P, 4, None, P, P, 1, 4), -1), ((two, 2, P, 4, None, None, P, 1, 4), -1), ((two, 2, P, 4, None, P, None, 1, 4), -1),
                         ((two, 2, None, 4, None, P, P, 1, 4), -1), ((two, 2, P, 4, None, P, P, 1, 257), -2), ((two, 2, P, 4, None, P, P, 65536, 4), -2), ((two, 2, P, 4, None, P, P, 0, 4), 0),
                         ((two, 2, P, 4, None, P, P, 1, 0), 0)):
        assert lib.et_kv_keep(*args, None) == status, args
    assert lib.et_kv_keep(two, 2, P, 4, None, P, P, 1, 4, None) == -1 and b"are the same" in lib.et_last_error()


def test_block_tables(et):
    def call(before=P, table=P, max_pages=4, page=16, npages=8, B=1, n=1, window=0, sinks=0, free=P, state=P, after=P, slots=None, ws=None, ws_bytes=0):
        return et.lib().et_kv_tables(before, table, max_pages, page, npages, None, None, None, B, n, window, sinks, free, state, after, slots, ws, ws_bytes, None)

    for bad, status in ((dict(before=None), -1), (dict(table=None), -1), (dict(free=None), -1), (dict(state=None), -1), (dict(after=None), -1), (dict(max_pages=0), -1), (dict(page=0), -1),
                        (dict(npages=0), -1), (dict(B=-1), -1), (dict(n=-1), -1), (dict(window=-1), -1), (dict(sinks=-1), -1), (dict(B=65536), -2), (dict(max_pages=1 << 28), -2),
                        (dict(B=4096, max_pages=1 << 20), -2), (dict(slots=P + 4), -2), (dict(B=600), -1), (dict(B=600, ws=P, ws_bytes=8), -1), (dict(B=600, ws=P + 4, ws_bytes=1 << 20), -2)):
        assert call(**bad) == status, bad
        assert et.lib().et_last_error().startswith(b"et_kv_tables:")
    assert et.kv_tables_workspace(4, 8) == 0 and et.kv_tables_workspace(8192, 512) > 0
    size = C.c_size_t()
    for args, status in (((0, 1, C.byref(size)), -1), ((4, -1, C.byref(size)), -1), ((4, 1, None), -1), ((4, 65536, C.byref(size)), -2)):
        assert et.lib().et_kv_tables_workspace(*args) == status


def test_the_oracle_of_tables_keeps_every_page_once():
    """Pages are in one table or in the ring, whatever comes and goes."""
    r = np.random.default_rng(1)
    B, M, page, npages, n = 5, 7, 4, 30, 9
    table, ring, state = np.full((B, M), -1, np.int32), r.permutation(npages).astype(np.int32), np.array([3, npages, 0], np.int32)
    for step in range(200):
        window, sinks = [(0, 0), (6, 0), (5, 3)][step % 3]
        starts, counts = r.integers(0, M * page - n, B), r.integers(0, n + 1, B)
        table, ring, state, slots = S.tables(table, page, npages, starts, counts, None, n, window, sinks, ring, state)
        held = table[table >= 0]
        free = ring[(state[0] + np.arange(state[1])) % npages]
        assert sorted([*held, *free]) == list(range(npages))
        got = slots[slots >= 0]
        assert len(set(got)) == len(got) and (state[2] > 0 or len(got) == counts.sum())
