"""Slots of many rows, which have a launch of their own behind the one that writes the tables: the rule, and the slots against plain loops."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

from oracle import sight as S
from tests.harness import up
from tests.test_gpu_tree import check_tables

ROOT = Path(__file__).resolve().parent.parent


def test_no_workgroup_has_many_slots(tmp_path):
    """However a call is made, a workgroup writes at most 3000 of them."""
    (tmp_path / "ask.cpp").write_text('#include <cstdio>\n#include "kv_tables_forms.h"\nint main() { int m, b, n; while (scanf("%d %d %d", &m, &b, &n) == 3) '
                                      'printf("%d %d\\n", (int)et::tables_of_one_workgroup(m, b), (int)et::slots_apart(m, b, n)); }\n')
    exe = tmp_path / "ask"
    subprocess.run(["g++", "-std=c++17", "-I", str(ROOT / "scpaper-2021_amd" / "csrc"), str(tmp_path / "ask.cpp"), "-o", str(exe)], check=True)
    sizes = [(m, b, n) for m in (1, 8, 64, 4096, 4097, 100000) for b in (1, 8, 64, 512, 513, 21474) for n in (0, 1, 6, 7, 48, 49, 512, 2048, 2049, 3000, 3001, (1 << 31) - 1)]
    out = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, s)) for s in sizes), capture_output=True, text=True, check=True).stdout.split("\n")
    for (m, b, n), line in zip(sizes, out):
        one, apart = map(int, line.split())
        assert one == (b <= 512 and b * m <= 4096)
        assert apart or (b * n if one else n) <= 3000
        assert not apart or (b * n if one else n) >= 2048


# (sequences, pages of each, tokens of a page, rows)
@pytest.mark.gpu
@pytest.mark.parametrize("B,M,page,n", [(8, 64, 16, 375), (8, 64, 16, 376), (512, 8, 128, 7), (512, 8, 128, 150), (1, 4096, 16, 5000), (1, 1, 16, 3100), (1, 5000, 16, 2048), (2, 5000, 16, 2049), (3, 2000, 4, 7999),
                                        (513, 8, 512, 2100)])
def test_slots_of_many_rows(et, B, M, page, n):
    r = np.random.default_rng(n)
    npages = max(4, B * M)
    before = np.where(r.random((B, M)) < 0.4, np.arange(B * M).reshape(B, M), -1).astype(np.int32)
    free = np.setdiff1d(np.arange(npages), before)
    ring = np.concatenate([free, np.full(npages - len(free), -7)]).astype(np.int32)
    for window, sinks in ((0, 0), (1000, 20)):
        starts, counts = r.integers(-5, max(1, M * page - n) + 20, B), r.integers(0, n + 2, B)
        check_tables(et, before, page, npages, starts, counts, None, n, window, sinks, ring, np.array([0, len(free) * 3 // 4, 0], np.int32), n % 2 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [40, 5000])
def test_recorded(et, M):
    """With the launch of the slots in a graph, replayed with starts that move on."""
    lib, B, page, n = et.lib(), 5, 16, 2100
    npages = B * M
    table, ring, state = np.full((B, M), -1, np.int32), np.arange(npages, dtype=np.int32), np.array([0, npages, 0], np.int32)
    dev, starts, counts = [up(et, a) for a in (table, ring, state)], up(et, np.zeros(B, np.int32)), up(et, np.zeros(B, np.int32))
    slots, need = up(et, np.zeros((B, n), np.int64)), et.kv_tables_workspace(M, B)
    ws = up(et, np.zeros(max(16, need), np.uint8))
    stream, graph = C.c_void_p(), C.c_void_p()
    et.check(lib.et_stream_create(C.byref(stream)))
    et.check(lib.et_graph_begin_capture(stream))
    et.kv_tables(dev[0], dev[0], M, page, npages, starts, counts, None, B, n, 300, 20, dev[1], dev[2], dev[2], slots, ws, need, stream)
    et.check(lib.et_graph_end_capture(stream, C.byref(graph)))
    r, at = np.random.default_rng(2), np.zeros(B, np.int32)
    for _ in range(5):
        now = r.integers(0, min(n, M * page // 6), B).astype(np.int32)
        for buf, a in ((starts, at), (counts, now)):
            et.check(lib.et_memcpy_h2d(buf.ptr, a.ctypes.data, a.nbytes))
        et.check(lib.et_graph_launch(graph, stream))
        et.check(lib.et_stream_sync(stream))
        table, ring, state, want = S.tables(table, page, npages, at, now, None, n, 300, 20, ring, state)
        for got, a in zip((*dev, slots), (table, ring, state, want)):
            assert np.array_equal(got.numpy(), a)
        at = (at + now).astype(np.int32)
    et.check(lib.et_graph_destroy(graph))
    et.check(lib.et_stream_destroy(stream))
