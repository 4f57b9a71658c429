"""Attention over a cache whose rows see a window and the first tokens, or the nodes of a tree, against binary64: every kernel that a call may run, at
sizes, windows and trees where it can go wrong.  Tolerances are those of attention over all keys (tests/test_gpu_kv_cache.py), derived there, since the sums are the
same over fewer keys; near results as a whole are held to 3e-4 of their 2-norm (tests/test_gpu_kv_precision.py)."""
import ctypes as C
import math

import numpy as np
import pytest

from oracle import decode as D
from oracle import sight as S
from tests import harness as Hn
from tests.harness import up
from tests.test_gpu_kv_cache import DeviceCache, allowed, filled, tables
from tests.test_gpu_kv_precision import NEAR, alternate, off, turning

pytestmark = pytest.mark.gpu


def trees(seed, B, n, back=8):
    """Parents of B trees: each node hangs on one of the few before it."""
    r = np.random.default_rng(seed)
    p = np.arange(n) - 1 - r.integers(0, back, (B, n))
    return np.where(np.arange(n) == 0, -1, np.maximum(p, 0)).astype(np.int32)


def run_window(et, dev, table, starts, counts, Q, B, n, nh, window, sinks, scale, causal, ldq=None, ldz=None, stream=None, workspace=None):
    width = nh * dev.host.hd
    ldq, ldz = ldq or width, ldz or width
    q = np.full((B * n, ldq), np.nan, np.float16)
    q[:, :width] = Q
    z = up(et, np.full((B * n, ldz), np.float16(-77)))
    need = et.mha_kv_window_workspace(dev.c, table.shape[1], B, n, nh, window, sinks)
    ws = workspace or up(et, np.full(max(need, 16), 0xFF, np.uint8))
    et.mha_kv_window(dev.c, up(et, table), table.shape[1], None if starts is None else up(et, np.array(starts, np.int32)), None if counts is None else up(et, np.array(counts, np.int32)),
                     up(et, q), ldq, z, ldz, B, n, nh, window, sinks, scale, et.MHA_CAUSAL if causal else 0, ws, need, stream)
    return z.numpy()


def run_tree(et, dev, table, starts, counts, words, Q, B, n, nh, window, sinks, scale, ldq=None, ldz=None):
    width = nh * dev.host.hd
    ldq, ldz = ldq or width, ldz or width
    q = np.full((B * n, ldq), np.nan, np.float16)
    q[:, :width] = Q
    z = up(et, np.full((B * n, ldz), np.float16(-77)))
    need = et.mha_kv_tree_workspace(dev.c, table.shape[1], B, n, nh, window, sinks)
    et.mha_kv_tree(dev.c, up(et, table), table.shape[1], up(et, np.array(starts, np.int32)), up(et, np.array(counts, np.int32)), up(et, words), up(et, q), ldq, z, ldz, B, n, nh,
                   window, sinks, scale, up(et, np.full(max(need, 16), 0xFF, np.uint8)), need)
    return z.numpy()


def gone(table, page, starts, window, sinks):
    """The table without the pages that no row sees any more; some of their entries name pages of others, or none."""
    table = table.copy()
    for b, s in enumerate(starts):
        for i in range(table.shape[1]):
            if i * page >= sinks and (i + 1) * page <= s - window + 1:
                table[b, i] = [-1, 99999, table[0, -1]][i % 3]
    return table


def near(got, Z, stepped, lows, reach, hd, keys, rows):
    """rows: of a key/value head.  Of more than 32, keys and values may enter the products as a binary16 number and what it leaves, at most half a step, 2^-11 of it, in 8 bits (e5m2, half a step
    is 2^-3), times a factor in 8 bits: off by 2^-11 (2^-3 + 2^-3 + 2^-6) = 1.3e-4 of a score's terms.  Of a value's that is as much, and what a weight leaves, in 8 bits, times the upper
    byte of the value (cut off: 2^-2): 2^-11 (2^-2 + 2^-3 + 2^-5) = 2.0e-4, in all 3.3e-4 of the sum of p |value|."""
    there = ~np.isnan(Z[:, 0])
    width = Z.shape[1]
    assert (got[:, width:] == -77).all() and (got[~there] == -77).all()
    d = np.abs(got[there, :width].astype(np.float64) - Z[there])
    lim = allowed(Z, stepped, lows, reach, hd, keys)[there]
    if rows > 32:
        lim += ((np.expm1(2 * 1.3e-4 * reach) + 3.3e-4) * (stepped + lows))[there]
    assert (d <= lim).all(), (np.nanmax(d / lim), np.argwhere(~(d <= lim))[:4])


def first(copies, got):
    """The rows of the first of several batches that are alike, each of which gives the same bits."""
    got = got.reshape(copies, -1, got.shape[-1])
    assert np.array_equal(got, np.broadcast_to(got[0], got.shape), equal_nan=True)
    return got[0]


def check_window(et, bits, nkv, per, hd, page, lengths, n, window, sinks, causal, seed=0, qscale=1.0, starts=None, ldq=None, ldz=None, more_pages=0, copies=1):
    B, nh = len(lengths), nkv * per
    max_pages = max(1, -(-max(lengths) // page)) + more_pages
    npages = B * max_pages + 1
    table = tables(seed + 1, B, max_pages, npages)
    host = filled(bits, nkv, hd, page, table, lengths, seed + 2, npages)
    starts = [l - min(n, l) for l in lengths] if starts is None else starts
    counts = [l - s for l, s in zip(lengths, starts)]
    Q = (np.random.default_rng(seed + 3).standard_normal((B * n, nh * hd)) * qscale).astype(np.float16)
    scale = 1 / math.sqrt(hd)
    got = first(copies, run_window(et, DeviceCache(et, host), np.tile(gone(table, page, starts, window, sinks), (copies, 1)), starts * copies, counts * copies, np.tile(Q, (copies, 1)), B * copies, n, nh,
                                   window, sinks, scale, causal, ldq, ldz))
    want = S.attention(host, table, starts, counts, Q, n, nh, scale, S.window_sight(starts, counts, n, window, sinks, causal))
    near(got, *want, hd, min(max(lengths), window + sinks + n), n * per)
    return got, want[0]


def check_tree(et, bits, nkv, per, hd, page, lengths, counts, n, window=0, sinks=0, seed=0, words=None, ldq=None, ldz=None, more_pages=0, copies=1):
    B, nh = len(lengths), nkv * per
    ends = [l + c for l, c in zip(lengths, counts)]
    max_pages = max(1, -(-max(ends) // page)) + more_pages
    npages = B * max_pages + 1
    table = tables(seed + 1, B, max_pages, npages)
    host = filled(bits, nkv, hd, page, table, ends, seed + 2, npages)
    if words is None:
        words = S.seen_words(trees(seed, B, n), counts, n)
    Q = np.random.default_rng(seed + 3).standard_normal((B * n, nh * hd)).astype(np.float16)
    scale = 1 / math.sqrt(hd)
    used = gone(table, page, lengths, window, sinks) if window else table
    got = first(copies, run_tree(et, DeviceCache(et, host), np.tile(used, (copies, 1)), lengths * copies, counts * copies, np.tile(words, (copies, 1, 1)), np.tile(Q, (copies, 1)), B * copies, n, nh, window,
                                 sinks, scale, ldq, ldz))
    want = S.attention(host, table, lengths, counts, Q, n, nh, scale, S.tree_sight(lengths, counts, n, words, window, sinks))
    near(got, *want, hd, max(ends), n * per)
    return got, want[0]


# (heads over each key/value head, rows): the kernels for one row, few rows, several and many
ROWS = [(1, 1), (4, 1), (2, 1), (3, 5), (1, 33), (4, 40)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("per,n", ROWS)
def test_window_head_sizes(et, bits, hd, per, n):
    check_window(et, bits, 2, per, hd, 16, [197, 1, 70], n, 50, 3, n > 1, seed=hd)


# many rows over a key/value head, and work for many workgroups
MANY = [(4, 40), (1, 130), (8, 33), (3, 100), (1, 256), (4, 10), (1, 64), (7, 7)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("per,n", MANY)
def test_window_many_rows(et, bits, hd, per, n):
    check_window(et, bits, 2, per, hd, 16, [497, 1, 70], n, 50, 3, True, seed=hd, copies=192)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("per,n", MANY)
def test_tree_many_rows(et, bits, hd, per, n):
    check_tree(et, bits, 2, per, hd, 16, [97, 0, 70], [n, n, max(1, n // 2)], n, seed=hd, copies=192)


@pytest.mark.parametrize("page", [16, 48, 64])
@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 16), (31, 1), (32, 33), (33, 0), (64, 100), (65, 5), (1 << 30, 0)])
def test_window_sizes_many_rows(et, page, window, sinks):
    for bits, hd, per, n, causal in ((4, 128, 8, 9, True), (8, 128, 4, 9, True), (8, 64, 1, 100, False), (4, 96, 2, 77, True), (8, 32, 3, 50, True)):
        check_window(et, bits, 1, per, hd, page, [300, 33, 64], n, window, sinks, causal, seed=page, copies=192)


@pytest.mark.parametrize("bits", [4, 8])
def test_many_rows_shared_out(et, bits):
    """Keys of many rows that several workgroups share: long contexts, and short ones beside tables for long ones."""
    check_tree(et, bits, 2, 4, 128, 64, [18000, 9], [30, 17], 30, seed=5)
    check_tree(et, bits, 4, 4, 128, 64, [3000, 9], [16, 7], 16, seed=11, more_pages=500)
    check_tree(et, bits, 8, 1, 128, 64, [9000, 30], [40, 40], 40, 8500, 20, seed=12, more_pages=3)
    check_tree(et, bits, 1, 1, 64, 48, [70, 0, 600], [130, 99, 1], 130, seed=6, more_pages=800)
    check_tree(et, bits, 6, 2, 96, 16, [9000, 30], [64, 64], 64, 8500, 20, seed=7, more_pages=3)
    check_window(et, bits, 4, 2, 128, 64, [9000, 200], 50, 8600, 70, True, seed=8)
    check_window(et, bits, 6, 3, 32, 16, [9000, 200], 50, 8600, 3, True, seed=9)
    check_window(et, bits, 6, 1, 64, 64, [9000, 200], 200, 8600, 3, True, seed=10, starts=[8800, 0])


def test_many_rows_strides(et):
    check_window(et, 4, 2, 2, 96, 16, [140, 85], 70, 60, 2, True, seed=8, ldq=3 * 384 + 8, ldz=384 + 8, copies=192)
    check_tree(et, 8, 2, 2, 128, 16, [140, 85], [70, 33], 70, seed=8, ldq=3 * 512 + 8, ldz=512 + 8, copies=64)
    check_tree(et, 4, 2, 2, 128, 16, [140, 85], [30, 13], 30, seed=8, ldq=3 * 512 + 8, ldz=512 + 8, copies=256)


def test_longest_first(et):
    """More workgroups than compute units, of sequences of every length: each its own rows."""
    r = np.random.default_rng(3)
    lengths = [int(x) for x in r.integers(0, 900, 40)]
    check_tree(et, 4, 8, 2, 128, 32, lengths, [int(x) for x in r.integers(0, 25, 40)], 24, seed=13)
    check_tree(et, 4, 8, 2, 128, 32, [90] * 40, [24] * 20 + [3] * 20, 24, seed=14, more_pages=20)


@pytest.mark.parametrize("page", [16, 48, 64])
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 64, 65, 200, 1 << 30])
@pytest.mark.parametrize("sinks", [0, 1, 16, 33, 100])
def test_window_sizes(et, page, window, sinks):
    check_window(et, 4, 1, 1, 64, page, [300, 33, 64], 1, window, sinks, False, seed=page)
    check_window(et, 4, 1, 2, 64, page, [300, 33, 64], 9, window, sinks, True, seed=page)
    check_window(et, 8, 1, 1, 128, page, [300, 33, 64], 3, window, sinks, False, seed=page)


@pytest.mark.parametrize("hd,per", [(64, 1), (128, 4), (256, 1), (32, 3)])
@pytest.mark.parametrize("causal", [False, True])
def test_window_of_a_piece_of_a_prompt(et, hd, per, causal):
    """More rows than the window holds, from position 0 on and later, and the last sequence short."""
    check_window(et, 4, 1, per, hd, 32, [150, 210, 20], 150, 40, 5, causal, seed=3, starts=[0, 60, 0])


@pytest.mark.parametrize("bits", [4, 8])
def test_window_shared_out(et, bits):
    """A window that several workgroups share; one sequence is shorter than it."""
    check_window(et, bits, 1, 4, 128, 64, [6000, 9], 1, 4000, 4, False, seed=5)
    check_window(et, bits, 2, 1, 64, 16, [5000, 3900], 2, 3333, 20, True, seed=6)
    check_window(et, bits, 1, 7, 96, 48, [5000, 9], 3, 4000, 70, True, seed=7)
    check_window(et, bits, 1, 8, 128, 64, [5000, 9], 40, 3800, 70, True, seed=8)


def test_window_strides_and_rows_that_see_nothing(et):
    check_window(et, 4, 2, 2, 96, 16, [140, 25], 3, 60, 2, True, seed=8, ldq=3 * 384 + 8, ldz=384 + 8)
    got, Z = check_window(et, 4, 2, 1, 64, 16, [3, 0, 20], 6, 4, 2, True, seed=3, starts=[-3, 0, 14])
    assert (Z[:3] == 0).all() and (got[:3] == 0).all()
    # the window lies on pages without a place, and nothing else is seen
    host = filled(4, 1, 64, 16, np.array([[0, 1, 2]], np.int32), [48], 1, 3)
    got = run_window(et, DeviceCache(et, host), np.array([[0, 1, -1]], np.int32), [47], [1], Hn.randn((1, 64), 1), 1, 1, 1, 9, 0, 0.1, False)
    assert (got == 0).all()


def test_window_behind_the_table(et):
    """Rows whose positions lie behind the last page see the first tokens and what is left of their window."""
    host = filled(4, 1, 64, 16, np.array([[0, 1]], np.int32), [32], 1, 2)
    dev, table, Q = DeviceCache(et, host), np.array([[0, 1]], np.int32), Hn.randn((2, 64), 1)
    for start in (30, 40, 2 ** 31 - 3):
        got = run_window(et, dev, table, [start], [2], Q, 1, 2, 1, 12, 3, 0.1, True)
        want = S.attention(host, table, [min(start, 60)], [2], Q, 2, 1, 0.1, S.window_sight([min(start, 60)], [2], 2, 12, 3, True))
        near(got, *want, 64, 32, 2)


@pytest.mark.parametrize("hd,per,n,copies", [(64, 1, 1, 1), (64, 1, 6, 1), (128, 2, 20, 1), (128, 1, 130, 512), (64, 1, 130, 1024), (128, 1, 40, 4000)])
def test_positions_beyond_32_bits(et, hd, per, n, copies):
    """Rows whose positions, and windows' beginnings, lie behind 2^31 see the first tokens alone; so do the nodes of a tree there."""
    host = filled(4, 1, hd, 16, np.array([[0, 1]], np.int32), [32], 1, 2)
    dev, table, Q = DeviceCache(et, host), np.tile(np.array([[0, 1]], np.int32), (copies, 1)), np.tile(Hn.randn((n, per * hd), 1), (copies, 1))
    words = np.tile(S.seen_words(np.arange(n, dtype=np.int32)[None] - 1, [n], n), (copies, 1, 1))
    for start in (2 ** 31 - 1, 2 ** 31 - 3):
        for window in (max(n, 2), 300):
            got = [run_window(et, dev, table, [start] * copies, [n] * copies, Q, copies, n, per, window, 3, 0.1, True),
                   run_tree(et, dev, table, [start] * copies, [n] * copies, words, Q, copies, n, per, window, 3, 0.1)]
            want = S.attention(host, table[:1], [1000], [n], Q[:n], n, per, 0.1, S.window_sight([1000], [n], n, window, 3, True))
            for z in got:
                near(first(copies, z), *want, hd, 32, n * per)


@pytest.mark.parametrize("hd,per,n", [(64, 1, 70), (128, 2, 60), (32, 3, 50)])
def test_starts_in_front_of_the_sequence(et, hd, per, n):
    """Rows in front of position 0 see nothing and become zero."""
    for copies in (1, 256):
        got, Z = check_window(et, 4, 1, per, hd, 16, [n - 30, 0, 14 + n], n, 20, 2, True, seed=3, starts=[-30, 0, 14], copies=copies)
        assert (Z[:30] == 0).all() and (got[:30] == 0).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("per,n", ROWS)
def test_tree_head_sizes(et, bits, hd, per, n):
    check_tree(et, bits, 2, per, hd, 16, [97, 0, 70], [n, n, max(1, n // 2)], n, seed=hd)


@pytest.mark.parametrize("n", [1, 2, 5, 31, 32, 33, 64, 65, 130, 256])
@pytest.mark.parametrize("page,lengths", [(16, [3, 31, 32]), (48, [33, 64, 95]), (64, [0, 1, 200])])
def test_tree_sizes(et, n, page, lengths):
    check_tree(et, 4, 1, 1, 64, page, lengths, [n, max(0, n - 1), n // 2], n, seed=page + n)


@pytest.mark.parametrize("hd,per,n,copies", [(64, 1, 1, 1), (64, 2, 1, 1), (64, 1, 20, 1), (128, 4, 9, 1), (256, 1, 3, 1), (32, 3, 40, 1), (128, 8, 33, 1), (128, 8, 33, 100), (128, 2, 20, 200), (64, 1, 100, 200), (32, 4, 40, 200)])
def test_tree_with_a_window(et, hd, per, n, copies):
    """Measured from a node's depth: the oldest keys that a node sees depend on how deep it is."""
    for window in (n, n + 1, 60, 300):
        check_tree(et, 4, 1, per, hd, 32, [280, 40, 0], [n, n, n], n, max(n, window), 5, seed=window, copies=copies)


@pytest.mark.parametrize("bits", [4, 8])
def test_tree_shared_out(et, bits):
    check_tree(et, bits, 1, 4, 128, 64, [5000, 9], [7, 3], 7, seed=5)
    check_tree(et, bits, 2, 1, 64, 16, [3333, 90], [64, 17], 64, seed=6)
    check_tree(et, bits, 1, 2, 96, 48, [6000, 90], [64, 17], 64, 4000, 7, seed=7)
    check_tree(et, bits, 1, 1, 64, 16, [4444], [1], 1, seed=8)


def test_tree_of_any_bits(et):
    """Rows of bits that are no tree's, a node that does not see itself, one that sees nothing, and bits of nodes that are not there."""
    r = np.random.default_rng(1)
    words = r.integers(0, 2 ** 32, (2, 40, 2), dtype=np.uint32)
    words[0, 3] = 0
    for per, hd, copies in ((1, 64, 1), (4, 128, 1), (1, 32, 1), (4, 128, 512), (1, 128, 1024), (4, 32, 512), (3, 64, 512), (3, 96, 512)):
        check_tree(et, 4, 1, per, hd, 16, [70, 0], [40, 23], 40, seed=2, words=words, copies=copies)
        check_tree(et, 4, 1, per, hd, 16, [70, 0], [40, 23], 40, 50, 3, seed=2, words=words, copies=copies)
    words[1, 0] = 0
    got, Z = check_tree(et, 4, 1, 1, 64, 16, [70, 0], [40, 23], 40, seed=2, words=words)
    assert (Z[40] == 0).all() and (got[40] == 0).all()


def test_tree_that_is_a_chain_is_causal_attention(et):
    """Bit for bit what attention up to the own position gives, by the same kernels."""
    for per, hd, n in ((1, 64, 1), (1, 64, 2), (3, 96, 5), (4, 128, 2)):
        B, lengths, nkv = 2, [75, 40], 2
        table = tables(1, B, 6, 12)
        host = filled(4, nkv, hd, 16, table, [l + n for l in lengths], 4, 12)
        dev, Q = DeviceCache(et, host), Hn.randn((B * n, nkv * per * hd), 5)
        words = S.seen_words(np.tile(np.arange(n, dtype=np.int32) - 1, (B, 1)), [n] * B, n)
        got = run_tree(et, dev, table, lengths, [n] * B, words, Q, B, n, nkv * per, 0, 0, 0.1)
        wide = run_window(et, dev, table, lengths, [n] * B, Q, B, n, nkv * per, 1 << 20, 0, 0.1, True)
        assert np.array_equal(got, wide)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd,per,n,copies", [(64, 1, 2, 1), (32, 1, 4, 1), (64, 3, 5, 1), (128, 1, 2, 1), (256, 2, 3, 1), (128, 4, 40, 1), (64, 1, 40, 1), (96, 2, 40, 1), (256, 1, 70, 1), (128, 4, 40, 64),
                                             (128, 4, 10, 256), (64, 1, 130, 128), (96, 2, 70, 128), (32, 4, 40, 128)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_not_a_number_where_others_look(et, bits, hd, per, n, copies, bad):
    """A node on nobody's way is NaN, and so are a token before the window and one between the first tokens and it: everyone else's rows are what they are without."""
    nkv, lengths = 2, [140, 64]
    nh, one = nkv * per, tables(1, 2, 20, 40)
    host = filled(bits, nkv, hd, 16, one, [l + n for l in lengths], 4, 40)
    table, B, lengths = np.tile(one, (copies, 1)), 2 * copies, lengths * copies
    Q = Hn.randn((B * n, nh * hd), 5)
    parents = np.tile(np.maximum(np.arange(n) - 1, 0), (B, 1)).astype(np.int32)
    parents[:, 0], parents[:, -1] = -1, max(0, n - 3)  # the last two are siblings, or the last is the root's child
    words = S.seen_words(parents, [n] * B, n)
    window, sinks = max(n, 50), 3
    tree = lambda: run_tree(et, DeviceCache(et, host), table, lengths, [n] * B, words, Q, B, n, nh, window, sinks, 0.1).reshape(B, n, -1)  # noqa: E731
    slide = lambda: run_window(et, DeviceCache(et, host), table, lengths, [n] * B, Q, B, n, nh, window, sinks, 0.1, True).reshape(B, n, -1)  # noqa: E731
    want, wide = tree(), slide()
    row = np.full((2, nkv * hd), bad, np.float16)
    for pos in ([sinks] * B, [sinks + 9] * B, [l - window for l in lengths]):
        host.write(one, pos[:2], [int(sinks <= p <= l - window) for p, l in zip(pos[:2], lengths)], row, row, 1)  # (a short sequence's window reaches to its beginning)
    assert np.array_equal(tree(), want) and np.array_equal(slide(), wide)
    if n > 1:
        host.write(one, [l + n - 1 for l in lengths[:2]], [1, 1], row, row, 1)
        got, last = tree(), slide()
        assert np.array_equal(got[:, :-1], want[:, :-1]) and np.isnan(got[:, -1]).all()
        assert np.array_equal(last[:, :-1], wide[:, :-1]) and np.isnan(last[:, -1]).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd,n", [(32, 130), (64, 130), (96, 130), (128, 130), (128, 50)])
def test_each_key_has_its_own_weight(et, bits, hd, n):
    """Of a sequence's values only one is not zero, 1, at another key for each sequence: the result is that key's weight, nothing at all for a row that does not see it."""
    B, page, length = 128, 16, 272
    table = np.hstack([tables(1, B, 17, B * 17), np.full((B, 60), -1, np.int32)])
    host = D.Cache(bits, 1, hd, page, B * 17)
    r = np.random.default_rng(1)
    K, V = r.standard_normal((length, hd)).astype(np.float16), np.zeros((B, length, hd), np.float16)
    V[np.arange(B), length - B + np.arange(B)] = 1
    host.write(table, [0] * B, [length] * B, np.tile(K, (B, 1)), V.reshape(-1, hd), length)
    Q = r.standard_normal((n, hd)).astype(np.float16)
    got = run_window(et, DeviceCache(et, host), table, [length - n] * B, [n] * B, np.tile(Q, (B, 1)), B, n, 1, 1 << 20, 0, 0.1, True).reshape(B, n, hd).astype(np.float64)
    score = np.where(np.arange(length) <= length - n + np.arange(n)[:, None], 0.1 * Q.astype(np.float64) @ D.stands_for(*D.quantise(K, 2 ** bits - 1)).T, -np.inf)
    p = np.exp(score - score.max(1, keepdims=True))
    p = (p / p.sum(1, keepdims=True))[:, length - B:].T[:, :, None]
    # a weight: half a step of the result; scores as for near(), their terms add up to less than 12 here
    assert (got[np.broadcast_to(p, got.shape) == 0] == 0).all() and (np.abs(got - p) <= (2.0 ** -11 + np.expm1(2 * 1.3e-4 * 12) + 2.0 ** -13) * p + 2.0 ** -25).all()


# (hd, key/value heads, query heads to each, rows, length, how many alike)
FORMS = [(32, 2, 1, 1, 300), (64, 2, 1, 1, 300), (128, 2, 1, 1, 300), (64, 2, 2, 1, 300), (128, 2, 4, 1, 300), (256, 2, 2, 1, 300), (64, 2, 5, 2, 300), (96, 2, 16, 1, 300), (128, 2, 3, 4, 300),
         (192, 2, 8, 1, 300), (256, 2, 8, 1, 300), (128, 2, 8, 1, 2100), (64, 2, 1, 40, 300), (128, 1, 8, 20, 300), (32, 1, 4, 40, 300), (64, 1, 1, 70, 5000), (96, 1, 3, 70, 700),
         (256, 1, 2, 70, 400), (160, 1, 4, 40, 300), (128, 1, 4, 64, 3500), (32, 1, 4, 40, 300, 320), (64, 1, 1, 130, 300, 320), (96, 1, 3, 70, 700, 200), (128, 1, 8, 20, 300, 160), (128, 1, 4, 16, 300, 480)]
LONG = [(128, 4, 1, 70, 20000)]  # many rows, keys shared out


def attended(et, bits, form, seed, qscale=1.0, values=lambda r, tokens, width: r.standard_normal((tokens, width)) * 0.5, keys=None):
    """(result, the same in binary64), [rows][heads][hd]: a window for odd seeds, a tree for even ones."""
    hd, nkv, per, n, length, copies = (*form, 1)[:6]
    r = np.random.default_rng(seed)
    width, nh = nkv * hd, nkv * per
    K = (r.standard_normal((length, width)) + 1.5 * r.standard_normal(width)).astype(np.float16)
    V = values(r, length, width).astype(np.float16)
    Q = r.standard_normal((n, nh * hd)) * qscale
    if keys:
        K, Q = keys(K, Q)
    Q = Q.astype(np.float16)
    page = 64
    max_pages = -(-length // page)
    table = tables(seed, 1, max_pages, max_pages)
    host = D.Cache(bits, nkv, hd, page, max_pages, fill=0xFF)
    host.write(table, [0], [length], K, V, length)
    starts, counts, dev, scale = [length - n], [n], DeviceCache(et, host), 1 / math.sqrt(hd)
    alike = lambda x: np.tile(x, (copies,) + (1,) * (np.ndim(x) - 1))  # noqa: E731
    if seed % 2:
        window, sinks = length // 2 + 11, 5
        got = run_window(et, dev, alike(table), alike(starts), alike(counts), alike(Q), copies, n, nh, window, sinks, scale, True)
        Z = S.attention(host, table, starts, counts, Q, n, nh, scale, S.window_sight(starts, counts, n, window, sinks, True))[0]
    else:
        words = S.seen_words(trees(seed, 1, n), counts, n)
        got = run_tree(et, dev, alike(table), alike(starts), alike(counts), alike(words), alike(Q), copies, n, nh, 0, 0, scale)
        Z = S.attention(host, table, starts, counts, Q, n, nh, scale, S.tree_sight(starts, counts, n, words, 0, 0))[0]
    return first(copies, got).astype(np.float64).reshape(-1, nh, hd), Z.reshape(-1, nh, hd)


def distance(got, Z):
    return np.linalg.norm(got - Z) / np.linalg.norm(Z)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("seed,qscale", [(11, 1.0), (12, 1.0), (13, 2.0 ** -13)])
@pytest.mark.parametrize("form", FORMS + LONG, ids=str)
def test_as_near_as_the_result_is_rounded(et, bits, form, seed, qscale):
    assert distance(*attended(et, bits, form, seed, qscale)) <= NEAR


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("every", [2, 7])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_values_of_single_tokens_far_larger(et, bits, form, every):
    assert distance(*attended(et, bits, form, 17, values=lambda r, tokens, width: r.standard_normal((tokens, width)) * np.where(np.arange(tokens) % every == every - 1, 128.0, 0.5)[:, None])) <= NEAR


def large_channel(K, Q):
    K[:, 2::32] = (K[:, 2::32] * 0.01).astype(np.float16)
    Q[:, 2::32] *= 200
    return K, Q


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("form", FORMS + LONG, ids=str)
def test_a_channel_far_larger_in_queries(et, bits, form):
    assert distance(*attended(et, bits, form, 18, keys=large_channel)) <= NEAR


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("qscale", [1.0, 2.0 ** -13])
@pytest.mark.parametrize("form", [f for f in FORMS if f[0] > 32], ids=str)
@pytest.mark.parametrize("values", [alternate(2.0 ** 13, 2.0 ** -7), turning(2.0 ** 13, 2.0 ** -7)], ids=["alternate", "turning"])
def test_groups_of_very_different_size(et, bits, form, qscale, values):
    """Channel groups whose values are 2^20 apart are each as near as if they were alone."""
    assert (off(*attended(et, bits, form, 21, qscale, values=values)) <= NEAR).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_keys_and_values_at_the_end_of_the_range(et, bits, form):
    """Groups from -65504 to 65504, whose scale's last steps lie beyond: keys against small queries, and values, which come out as the largest number at most."""
    got, Z = attended(et, bits, form, 13, qscale=2.0 ** -17, values=lambda r, tokens, width: np.tile(np.where(np.arange(width) % 3, 65504.0, -65504.0), (tokens, 1)),
                      keys=lambda K, Q: (np.where(K > 0, np.float16(65504), np.float16(-65504)), Q))
    want = np.clip(Z, -65504, 65504)
    assert np.isfinite(got).all() and (np.abs(got - want) <= 2.0 ** -10 * np.abs(want)).all()


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("seed", [14, 15])
def test_infinite_queries_make_their_row_not_a_number(et, form, bad, seed):
    def put(K, Q):
        Q[0, 5] = bad
        return np.abs(K) + np.float16(1), Q
    with np.errstate(invalid="ignore"):
        got, _ = attended(et, 4, form, seed, keys=put)
    want, _ = attended(et, 4, form, seed, keys=lambda K, Q: (np.abs(K) + np.float16(1), Q))
    assert np.isnan(got[0, 0]).all()
    got[0, 0] = want[0, 0]
    assert np.array_equal(got, want)


def test_large_offsets(et):
    """A cache whose last pages lie beyond 2^32 bytes: the table names only those."""
    nkv, hd, page = 16, 256, 128
    npages = (1 << 32) // (nkv * hd // 2 * page) + 3
    codes = [et.DeviceBuffer(npages * nkv * hd // 2 * page) for _ in range(2)]
    scales = [et.DeviceBuffer(npages * nkv * 8 * page * 4) for _ in range(2)]
    c = et.KvCache(codes[0].ptr, scales[0].ptr, codes[1].ptr, scales[1].ptr, 4, nkv, hd, page, npages)
    length = 200
    K, V = Hn.randn((length, nkv * hd), 1), Hn.randn((length, nkv * hd), 2)
    d_table = up(et, np.array([[npages - 1, npages - 3]], np.int32))
    et.kv_write(c, d_table, 2, None, None, up(et, K), up(et, V), nkv * hd, nkv * hd, 1, length)
    table = np.array([[0, 1]], np.int32)
    host = D.Cache(4, nkv, hd, page, 2)
    host.write(table, [0], [length], K, V, length)
    for n in (1, 40):
        Q, z = Hn.randn((n, nkv * hd), 3), up(et, np.zeros((n, nkv * hd), np.float16))
        need = et.mha_kv_window_workspace(c, 2, 1, n, nkv, 90, 4)
        et.mha_kv_window(c, d_table, 2, up(et, np.array([length - n], np.int32)), None, up(et, Q), nkv * hd, z, nkv * hd, 1, n, nkv, 90, 4, 1 / 16, et.MHA_CAUSAL,
                         up(et, np.zeros(max(need, 16), np.uint8)), need)
        near(z.numpy(), *S.attention(host, table, [length - n], [n], Q, n, nkv, 1 / 16, S.window_sight([length - n], [n], n, 90, 4, True)), hd, length, n)
    # the path moves there, too: the last token to where the second stands
    path, kept = up(et, np.array([[0, length - 1]], np.int32)), up(et, np.array([2], np.int32))
    start = up(et, np.array([0], np.int32))
    et.kv_keep([c], d_table, 2, start, path.ptr, kept, 1, 2)  # 199 is no row of two: left out
    k, v = (up(et, np.zeros((length, nkv * hd), np.float16)) for _ in range(2))
    et.kv_read(c, d_table, 2, None, None, k, v, nkv * hd, nkv * hd, 1, length)
    assert np.array_equal(k.numpy(), D.to_f16(D.stands_for(*D.quantise(K, 15)))) and np.array_equal(v.numpy(), D.to_f16(D.stands_for(*D.quantise(V, 15))))
    moved = np.r_[0, 170, np.arange(2, length)]
    et.kv_keep([c], d_table, 2, start, up(et, np.array([[0, 170] + [-1] * 198], np.int32)), kept, 1, 200)
    et.kv_read(c, d_table, 2, None, None, k, v, nkv * hd, nkv * hd, 1, length)
    assert np.array_equal(k.numpy(), D.to_f16(D.stands_for(*D.quantise(K[moved], 15)))) and np.array_equal(v.numpy(), D.to_f16(D.stands_for(*D.quantise(V[moved], 15))))


def test_on_two_streams_at_once_and_again(et):
    """Two batches over one cache, keys shared out over workgroups, each with its stream and workspace: the bits that each gives alone, however often."""
    lib = et.lib()
    table = tables(2, 2, 300, 600)
    host = filled(4, 2, 64, 16, table, [4600, 900], 7, 600)
    dev = DeviceCache(et, host)
    dt, ds = up(et, table), up(et, np.array([4599, 899], np.int32))
    Q = [Hn.randn((2, 256), 5), Hn.randn((2, 256), 6)]
    want = [run_window(et, dev, table, [4599, 899], None, q, 2, 1, 4, 4000, 5, 0.125, False) for q in Q]
    need = et.mha_kv_window_workspace(dev.c, 300, 2, 1, 4, 4000, 5)
    assert need > 0
    streams, q, z, ws = [], [up(et, x) for x in Q], [], []
    for _ in Q:
        s = C.c_void_p()
        et.check(lib.et_stream_create(C.byref(s)))
        streams.append(s)
        z.append(up(et, np.zeros((20, 2, 256), np.float16)))
        ws.append(up(et, np.full(need, 0xFF, np.uint8)))
    for i in range(20):
        for k, s in enumerate(streams):
            et.mha_kv_window(dev.c, dt, 300, ds, None, q[k], 256, z[k].offset(i * 2 * 256 * 2), 256, 2, 1, 4, 4000, 5, 0.125, 0, ws[k], need, s)
    for k, s in enumerate(streams):
        et.check(lib.et_stream_sync(s))
        assert (z[k].numpy() == want[k]).all()
        et.check(lib.et_stream_destroy(s))


@pytest.mark.parametrize("hd,per,n,length", [(128, 2, 60, 3000), (128, 4, 16, 8200), (64, 2, 100, 6500), (128, 1, 16, 3000)])
def test_many_rows_recorded_on_two_streams(et, hd, per, n, length):
    """Keys shared out over workgroups, without starts or counts: two graphs of a window's and a tree's attention, each with its workspace, replayed side by side, and the bits of eager calls each time."""
    lib, nkv, B, page = et.lib(), 8, 2, 64
    pages = -(-length // page)
    table = tables(2, B, pages, B * pages)
    host = filled(4, nkv, hd, page, table, [length] * B, 7, B * pages)
    dev, width, dt = DeviceCache(et, host), nkv * per * hd, up(et, table)
    starts = up(et, np.full(B, length - n, np.int32))
    words = up(et, S.seen_words(trees(3, B, n), [n] * B, n))
    q = [up(et, Hn.randn((B * n, width), 5 + k)) for k in range(2)]
    need = [et.mha_kv_tree_workspace(dev.c, pages, B, n, nkv * per, 0, 0), et.mha_kv_window_workspace(dev.c, pages, B, n, nkv * per, length - 200, 7)]
    assert min(need) > 0 or n * per <= 32

    def run(k, z, ws, stream):
        if k == 0:
            et.mha_kv_tree(dev.c, dt, pages, starts, None, words, q[0], width, z, width, B, n, nkv * per, 0, 0, 0.1, ws, need[0], stream)
        else:
            et.mha_kv_window(dev.c, dt, pages, starts, None, q[1], width, z, width, B, n, nkv * per, length - 200, 7, 0.1, et.MHA_CAUSAL, ws, need[1], stream)

    new = lambda k: (up(et, np.zeros((B * n, width), np.float16)), up(et, np.full(max(need[k], 16), 0xFF, np.uint8)))  # noqa: E731
    want, streams, graphs, out = [], [], [], []
    for k in range(2):
        z, ws = new(k)
        run(k, z, ws, None)
        et.check(lib.et_device_sync())
        want.append(z.numpy())
        out.append(new(k))
        s, g = C.c_void_p(), C.c_void_p()
        et.check(lib.et_stream_create(C.byref(s)))
        et.check(lib.et_graph_begin_capture(s))
        run(k, *out[k], s)
        et.check(lib.et_graph_end_capture(s, C.byref(g)))
        streams.append(s)
        graphs.append(g)
    for _ in range(6):
        for k in range(2):
            zero = np.zeros((B * n, width), np.float16)
            et.check(lib.et_memcpy_h2d(out[k][0].ptr, zero.ctypes.data, zero.nbytes))
            et.check(lib.et_graph_launch(graphs[k], streams[k]))
        run(0, *(eager := new(0)), None)
        et.check(lib.et_device_sync())
        assert np.array_equal(eager[0].numpy(), want[0])
        for k in range(2):
            assert np.array_equal(out[k][0].numpy(), want[k])
    for g, s in zip(graphs, streams):
        et.check(lib.et_graph_destroy(g))
        et.check(lib.et_stream_destroy(s))
    # from position 0 on, and n rows of each sequence
    z, ws = new(1)
    et.mha_kv_window(dev.c, dt, pages, None, None, q[1], width, z, width, B, n, nkv * per, 40, 3, 0.1, et.MHA_CAUSAL, ws, need[1], None)
    near(z.numpy(), *S.attention(host, table, [0] * B, [n] * B, q[1].numpy(), n, nkv * per, 0.1, S.window_sight([0] * B, [n] * B, n, 40, 3, True)), hd, n, n * per)
