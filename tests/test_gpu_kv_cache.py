"""The paged cache of keys and values in 4 and 8 bits: what et_kv_write_f16 stores is compared bit for bit with the format
built in numpy, on buffers that hold a pattern before (so a byte written beside its place shows), and what et_kv_read_f16 gives with what
the codes stand for; attention over the cache against binary64."""
import ctypes as C
import math

import numpy as np
import pytest

from oracle import decode as D
from tests import harness as Hn
from tests.harness import up

pytestmark = pytest.mark.gpu


class DeviceCache:
    """A host cache and its copy on the device."""

    def __init__(self, et, host):
        self.et, self.host = et, host
        self.bufs = {k: up(et, getattr(host, k)) for k in ("k_codes", "k_scales", "v_codes", "v_scales")}
        self.c = et.KvCache(*(self.bufs[k].ptr for k in ("k_codes", "k_scales", "v_codes", "v_scales")), host.bits, host.nkv, host.hd, host.page, host.npages)

    def same(self):
        for k, buf in self.bufs.items():
            got, want = buf.numpy(), getattr(self.host, k)
            if got.dtype == np.float16:
                # a NaN for a NaN; else the same number (a lowest value of zero has either sign)
                assert np.array_equal(np.isnan(got), np.isnan(want)), k
                got, want = np.nan_to_num(got, posinf=np.inf, neginf=-np.inf), np.nan_to_num(want, posinf=np.inf, neginf=-np.inf)
            assert np.array_equal(got, want), (k, np.argwhere(got != want)[:5])


def tables(seed, B, max_pages, npages):
    return np.random.default_rng(seed).permutation(npages)[:B * max_pages].reshape(B, max_pages).astype(np.int32)


def hard_values(shape, seed):
    """Binary16 values of many kinds of groups of 32: ordinary, far from zero, on the borders of steps, subnormal, equal, over the whole range."""
    r = np.random.default_rng(seed)
    x = r.standard_normal((int(np.prod(shape)) // 32, 32))
    kind = np.arange(len(x)) % 8
    x[kind == 1] = x[kind == 1] * 0.25 + 40
    x[kind == 2] = r.integers(0, 31, x[kind == 2].shape) * 0.5 + 3         # halves of a scale of 1
    x[kind == 2, 0], x[kind == 2, 1] = 3, 18
    x[kind == 3] = r.integers(-40, 41, x[kind == 3].shape) * 2.0 ** -24
    x[kind == 4] = x[kind == 4][:, :1]
    x[kind == 5] = r.choice([-65504.0, 65504.0, 1.0, -3.0, 2.0 ** -24, 0.0], x[kind == 5].shape)
    x[kind == 6] = np.exp2(r.uniform(-24, 15, x[kind == 6].shape)) * r.choice([-1, 1], x[kind == 6].shape)
    return x.astype(np.float16).reshape(shape)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("nkv,hd,page,B,n,starts,counts", [
    (1, 32, 16, 1, 1, [0], [1]),
    (12, 64, 16, 3, 1, [5, 15, 16], [1, 1, 1]),
    (3, 96, 48, 2, 70, [0, 45], [70, 33]),
    (2, 128, 32, 4, 9, [3, 0, 30, 61], [9, 0, 2, 9]),
    (1, 256, 16, 2, 37, [14, 1], [37, 36]),
    (2, 160, 128, 1, 130, [127], [130]),
    (5, 224, 16, 2, 5, [-3, 78], [5, 5]),        # rows before the first position, and behind the last page
    (4, 192, 64, 3, 6, [2, 3, 1], [100, -1, 6]),  # counts beyond what there is
])
def test_write_and_read(et, bits, nkv, hd, page, B, n, starts, counts):
    width, max_pages = nkv * hd, 5 if hd == 224 else -(-(max(starts) + n) // page)
    npages = B * max_pages + 2
    host = D.Cache(bits, nkv, hd, page, npages)
    table = tables(1, B, max_pages, npages)
    ldk, ldv = width + 8, 2 * width
    K, V = hard_values((B * n, width), 2), hard_values((B * n, width), 3)[::-1].copy()
    rows_k, rows_v = np.full((B * n, ldk), np.nan, np.float16), np.full((B * n, ldv), np.nan, np.float16)
    rows_k[:, :width], rows_v[:, :width] = K, V
    dev = DeviceCache(et, host)
    s, c = np.array(starts, np.int32), np.array(counts, np.int32)
    where = (dev.c, up(et, table).ptr, max_pages, up(et, s).ptr, up(et, c).ptr)
    et.kv_write(*where, up(et, rows_k), up(et, rows_v), ldk, ldv, B, n)
    host.write(table, s, c, K, V, n)
    dev.same()

    marker = np.float16(-1234)
    for which in ("both", "k", "v"):
        k, v = np.full((B * n, ldk), marker), np.full((B * n, ldv), marker)
        dk, dv = up(et, k), up(et, v)
        et.kv_read(*where, dk if which != "v" else None, dv if which != "k" else None, ldk, ldv, B, n)
        for b in range(B):
            for i in range(min(max(counts[b], 0), n)):
                at = host.place(table, b, starts[b] + i)
                if at is not None:
                    tok = [D.to_f16(D.stands_for(*t)).reshape(-1) for t in host.token(*at)]
                    if which != "v":
                        k[b * n + i, :width] = tok[0]
                    if which != "k":
                        v[b * n + i, :width] = tok[1]
        assert np.array_equal(dk.numpy(), k) and np.array_equal(dv.numpy(), v), which
    dev.same()


@pytest.mark.parametrize("bits", [4, 8])
def test_not_a_number_stays_in_its_group(et, bits):
    host = D.Cache(bits, 1, 64, 16, 2)
    K, V = Hn.randn((6, 64), 1), Hn.randn((6, 64), 2)
    K[1, 3], K[2, 40], V[4, 63], V[0, 0] = np.nan, np.inf, -np.inf, np.nan
    dev = DeviceCache(et, host)
    table, s, c = np.array([[1]], np.int32), np.array([4], np.int32), np.array([6], np.int32)
    where = (dev.c, up(et, table).ptr, 1, up(et, s).ptr, up(et, c).ptr)
    et.kv_write(*where, up(et, K), up(et, V), 64, 64, 1, 6)
    host.write(table, s, c, K, V, 6)
    dev.same()
    dk, dv = up(et, np.zeros((6, 64), np.float16)), up(et, np.zeros((6, 64), np.float16))
    et.kv_read(*where, dk, dv, 64, 64, 1, 6)
    nan = np.zeros((2, 6, 2), bool)
    nan[0, 1, 0] = nan[0, 2, 1] = nan[1, 4, 1] = nan[1, 0, 0] = True
    assert np.array_equal(np.isnan(np.stack([dk.numpy(), dv.numpy()])).reshape(2, 6, 2, 32).all(-1), nan)
    assert np.isnan(np.stack([dk.numpy(), dv.numpy()])).sum() == 4 * 32


@pytest.mark.parametrize("bits", [4, 8])
def test_token_by_token_equals_all_at_once(et, bits):
    """Also without starts and counts, and with pages that have no place among them."""
    host = D.Cache(bits, 2, 64, 16, 5)
    n = 45
    K, V = Hn.randn((n, 128), 3), Hn.randn((n, 128), 4)
    table = np.array([[4, -1, 1]], np.int32)
    dev, dev2 = DeviceCache(et, host), DeviceCache(et, D.Cache(bits, 2, 64, 16, 5))
    dt = up(et, table)
    et.kv_write(dev.c, dt, 3, None, None, up(et, K), up(et, V), 128, 128, 1, n)
    dk, dv = up(et, K), up(et, V)
    steps = [up(et, np.array([i], np.int32)) for i in range(n)]
    for i in range(n):
        et.kv_write(dev2.c, dt, 3, steps[i], None, dk.offset(i * 256), dv.offset(i * 256), 128, 128, 1, 1)
    host.write(table, [0], [n], K, V, n)
    dev.same()
    dev2.host = host
    dev2.same()
    table = np.array([[4, 5, 1]], np.int32)  # page 5 of 5
    et.kv_write(dev.c, up(et, table), 3, None, None, up(et, K), up(et, V), 128, 128, 1, n)
    dev.same()


# ---- attention -----------------------------------------------------------------------------------------------

def allowed(Z, stepped, lows, reach, hd, keys):
    """How far a row of et_mha_kv_f16 may be from binary64.  Half a step of binary16 (2^-11, relative) for the result and for every
    probability times scale; scores off by d, from hd + 16 roundings of 2^-24 in sums of magnitude `reach` and 2^-20 for exp2, move every p by
    d, and the sum of p by d; sums over the keys are in binary32 (keys + 16 roundings of 2^-24).  A product of probability and scale that is a
    subnormal binary16 number is off by half a step of those instead, 2^-25, where the largest stands between 2^10 and 2^15 and the values
    reach over at most 8 (they lie within 4 of zero): 2^-35 * 8 a key.  A subnormal result: 2^-25."""
    d = (hd + 16) * 2.0 ** -24 * reach + 2.0 ** -20
    a = stepped + lows
    return 2.0 ** -11 * np.abs(Z) + 2.0 ** -11 * stepped * (1 + 2.0 ** -10) + (2 * np.expm1(2 * d) + (keys + 16) * 2.0 ** -24) * a + keys * 2.0 ** -32 + 2.0 ** -25


def filled(bits, nkv, hd, page, table, lengths, seed, npages):
    """A cache with `lengths` tokens of random keys and values; everything else in it is NaN."""
    host = D.Cache(bits, nkv, hd, page, npages, fill=0xFF)
    B, n = len(lengths), max(max(lengths), 1)
    r = np.random.default_rng(seed)
    K = (r.standard_normal((B * n, nkv * hd)) + 1.5 * r.standard_normal(nkv * hd)).astype(np.float16)
    V = (r.standard_normal((B * n, nkv * hd)) * 0.5).astype(np.float16)
    host.write(table, [0] * B, lengths, K, V, n)
    return host


def run_attention(et, dev, table, starts, counts, Q, B, n, nh, scale, causal, ldq=None, ldz=None, stream=None):
    hd = dev.host.hd
    width = nh * hd
    ldq, ldz = ldq or width, ldz or width
    q = np.full((B * n, ldq), np.nan, np.float16)
    q[:, :width] = Q
    z = up(et, np.full((B * n, ldz), np.float16(-77)))
    need = et.mha_kv_workspace(dev.c, table.shape[1], B, n, nh)
    ws = up(et, np.full(max(need, 16), 0xFF, np.uint8))
    et.mha_kv(dev.c, up(et, table), table.shape[1], None if starts is None else up(et, np.array(starts, np.int32)),
              None if counts is None else up(et, np.array(counts, np.int32)), up(et, q), ldq, z, ldz, B, n, nh, scale, et.MHA_CAUSAL if causal else 0, ws, need, stream)
    return z.numpy()


def check_attention(et, bits, nkv, per, hd, page, lengths, n, causal, seed=0, qscale=1.0, starts=None, ldq=None, ldz=None, table=None, scale=None):
    B, nh = len(lengths), nkv * per
    max_pages = max(1, -(-max(lengths) // page))
    npages = B * max_pages + 1
    table = tables(seed + 1, B, max_pages, npages) if table is None else table
    host = filled(bits, nkv, hd, page, table, lengths, seed + 2, npages)
    starts = [l - min(n, l) for l in lengths] if starts is None else starts
    counts = [l - s for l, s in zip(lengths, starts)]
    Q = (np.random.default_rng(seed + 3).standard_normal((B * n, nh * hd)) * qscale).astype(np.float16)
    scale = 1 / math.sqrt(hd) if scale is None else scale
    got = run_attention(et, DeviceCache(et, host), table, starts, counts, Q, B, n, nh, scale, causal, ldq, ldz)
    Z, stepped, lows, reach = D.attention(host, table, starts, counts, Q, n, nh, scale, causal)
    width = nh * hd
    there = ~np.isnan(Z[:, 0])
    assert (got[:, width:] == -77).all() and (got[~there] == -77).all()
    off = np.abs(got[there, :width].astype(np.float64) - Z[there])
    lim = allowed(Z, stepped, lows, reach, hd, max(lengths))[there]
    assert (off <= lim).all(), (np.nanmax(off / lim), np.argwhere(~(off <= lim))[:4])
    return got, Z


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("per,n,causal", [(1, 1, False), (4, 1, False), (3, 5, True)])
def test_attention_head_sizes(et, bits, hd, per, n, causal):
    check_attention(et, bits, 2, per, hd, 16, [67, 1, 40], n, causal, seed=hd)


@pytest.mark.parametrize("page", [16, 48, 64, 128])
@pytest.mark.parametrize("lengths", [[1], [15, 16, 17], [31, 32, 33], [63, 64, 65, 127], [257, 3], [700]])
def test_attention_lengths(et, page, lengths):
    check_attention(et, 4, 2, 1, 64, page, lengths, 1, False, seed=page)


@pytest.mark.parametrize("per,n,nkv", [(1, 2, 3), (2, 1, 2), (5, 1, 1), (8, 1, 2), (16, 1, 1), (16, 3, 1), (8, 9, 1), (1, 33, 2), (7, 16, 1), (64, 1, 1)])
@pytest.mark.parametrize("hd,causal", [(64, True), (128, False)])
def test_attention_rows(et, per, n, nkv, hd, causal):
    check_attention(et, 4, nkv, per, hd, 32, [90, 40, 7], n, causal, seed=per + n)


@pytest.mark.parametrize("bits", [4, 8])
def test_attention_long(et, bits):
    """Sequences that are shared out over many workgroups, one of them short."""
    check_attention(et, bits, 1, 4, 128, 64, [5000, 9], 1, False, seed=5)
    check_attention(et, bits, 2, 1, 64, 16, [3333], 2, True, seed=6)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd", [64, 96, 256])
def test_attention_long_of_many_rows(et, bits, hd):
    """Many rows a key/value head over keys that are shared out: the last block of rows is not full, one sequence has no key for most workgroups."""
    check_attention(et, bits, 1, 7, hd, 48, [4000, 9], 3, True, seed=15)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("lengths,nkv,per,n", [([2100, 40], 3, 8, 1), ([2049, 9], 1, 1, 7), ([40] * 86, 3, 5, 1), ([33] * 64, 4, 2, 3), ([5000], 1, 3, 2)])
def test_attention_five_to_eight_rows(et, bits, lengths, nkv, per, n):
    """Heads of 128: blocks of 8 rows where there are many heads, or long sequences."""
    check_attention(et, bits, nkv, per, 128, 64, lengths, n, True, seed=21)


@pytest.mark.parametrize("bits", [4, 8])
def test_attention_not_a_number_of_a_later_token_in_blocks_of_eight(et, bits):
    lengths, n, nkv = [2060, 30], 5, 2
    table = tables(1, 2, 33, 66)
    host = filled(bits, nkv, 128, 64, table, lengths, 4, 66)
    starts = [l - n for l in lengths]
    Q = Hn.randn((2 * n, nkv * 128), 5)
    want = run_attention(et, DeviceCache(et, host), table, starts, None, Q, 2, n, nkv, 0.125, True).reshape(2, n, -1)
    row = np.full((2, nkv * 128), np.nan, np.float16)
    host.write(table, [l - 1 for l in lengths], [1] * 2, np.ones_like(row), row, 1)
    got = run_attention(et, DeviceCache(et, host), table, starts, None, Q, 2, n, nkv, 0.125, True).reshape(2, n, -1)
    assert np.array_equal(got[:, :-1], want[:, :-1]) and np.isnan(got[:, -1]).all()


@pytest.mark.parametrize("qscale", [2.0 ** -13, 30.0])
def test_attention_of_very_even_and_very_uneven_probabilities(et, qscale):
    check_attention(et, 4, 2, 2, 64, 16, [300, 81], 1, False, seed=9, qscale=qscale)
    check_attention(et, 8, 1, 1, 128, 16, [300], 1, False, seed=9, qscale=qscale)


def test_attention_scale_of_either_sign_and_zero(et):
    for scale in (-0.2, 0.0):
        check_attention(et, 4, 1, 2, 64, 16, [70], 1, False, seed=4, scale=scale)


def test_attention_rows_that_see_nothing(et):
    """Empty sequences, rows in front of the first position, and pages without a place: zero, and no NaN of the cache's rest."""
    got, Z = check_attention(et, 4, 2, 1, 64, 16, [3, 0, 20], 6, True, seed=3, starts=[-3, 0, 14])
    assert (Z[:3] == 0).all() and (got[:3] == 0).all()
    got, Z = check_attention(et, 4, 2, 1, 64, 16, [40, 16], 1, False, seed=3, table=np.array([[2, -1, 9999], [-5, 0, 1]], np.int32))
    assert (Z[1] == 0).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd,per,n", [(64, 1, 2), (32, 1, 4), (32, 1, 3), (64, 3, 5), (128, 1, 2), (256, 2, 3)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_attention_not_a_number_of_a_later_token(et, bits, hd, per, n, bad):
    """The last token's key and value are NaN, which with causal attention only its own row sees: the other rows are what they are without it."""
    nkv, lengths = 2, [40, n, 64 + n]
    B, nh = len(lengths), nkv * per
    table = tables(1, B, 5, 15)
    host = filled(bits, nkv, hd, 16, table, lengths, 4, 15)
    starts = [l - n for l in lengths]
    Q = Hn.randn((B * n, nh * hd), 5)
    want = run_attention(et, DeviceCache(et, host), table, starts, None, Q, B, n, nh, 0.125, True)
    row = np.full((B, nkv * hd), bad, np.float16)
    for K, V in ((row, row), (np.ones_like(row), row)):
        host.write(table, [l - 1 for l in lengths], [1] * B, K, V, 1)
        got = run_attention(et, DeviceCache(et, host), table, starts, None, Q, B, n, nh, 0.125, True).reshape(B, n, -1)
        assert np.array_equal(got[:, :-1], want.reshape(B, n, -1)[:, :-1])
        assert np.isnan(got[:, -1]).all()


def test_attention_strides(et):
    check_attention(et, 4, 2, 2, 96, 16, [40, 25], 3, True, seed=8, ldq=3 * 384 + 8, ldz=384 + 8)


def test_attention_without_starts_and_counts_is_self_attention(et):
    """n rows from position 0 on: what et_mha_fused_f16 computes on the values that the cache stands for."""
    B, n, nh, hd = 2, 48, 3, 64
    K, V, Q = (Hn.randn((B * n, nh * hd), s) for s in (1, 2, 3))
    dev = DeviceCache(et, D.Cache(4, nh, hd, 16, 6))
    dt = up(et, np.arange(6, dtype=np.int32).reshape(2, 3))
    et.kv_write(dev.c, dt, 3, None, None, up(et, K), up(et, V), nh * hd, nh * hd, B, n)
    k, v, z, want = (up(et, np.zeros((B * n, nh * hd), np.float16)) for _ in range(4))
    et.kv_read(dev.c, dt, 3, None, None, k, v, nh * hd, nh * hd, B, n)
    need = et.mha_kv_workspace(dev.c, 3, B, n, nh)
    dq = up(et, Q)
    for causal in (0, et.MHA_CAUSAL):
        et.mha_kv(dev.c, dt, 3, None, None, dq, nh * hd, z, nh * hd, B, n, nh, 0.125, causal, up(et, np.zeros(max(need, 16), np.uint8)), need)
        et.mha_fused(dq, k, v, nh * hd, nh * hd, nh * hd, want, nh * hd, None, None, B, n, nh, hd, 0.125, causal)
        # reading back rounds every channel of a key by up to 2^-11: scores are off by d, probabilities by twice d and 2^-11; then values and results
        q, key, top = np.abs(Q.astype(np.float64)).reshape(B, n, nh, hd), np.abs(k.numpy().astype(np.float64)).reshape(B, n, nh, hd), np.abs(v.numpy()).max()
        d = 2.0 ** -11 * 0.125 * np.einsum("bihd,bjhd->bhij", q, key).max()
        assert Hn.max_abs(z.numpy(), want.numpy()) <= (2 * np.expm1(2 * d) + 6 * 2.0 ** -11) * top


def test_attention_takes_large_offsets(et):
    """A cache whose last pages lie beyond 2^32 bytes: the table names only those."""
    nkv, hd, page = 16, 256, 128
    token = nkv * hd // 2 * page
    npages = (1 << 32) // token + 3
    codes = [et.DeviceBuffer(npages * token) for _ in range(2)]
    scales = [et.DeviceBuffer(npages * nkv * 8 * page * 4) for _ in range(2)]
    c = et.KvCache(codes[0].ptr, scales[0].ptr, codes[1].ptr, scales[1].ptr, 4, nkv, hd, page, npages)
    n = 200
    K, V = Hn.randn((n, nkv * hd), 1), Hn.randn((n, nkv * hd), 2)
    table = up(et, np.array([[npages - 1, npages - 3]], np.int32))
    et.kv_write(c, table, 2, None, None, up(et, K), up(et, V), nkv * hd, nkv * hd, 1, n)
    host = D.Cache(4, nkv, hd, page, 2)
    host.write(np.array([[0, 1]], np.int32), [0], [n], K, V, n)
    k, v = (up(et, np.zeros((n, nkv * hd), np.float16)) for _ in range(2))
    et.kv_read(c, table, 2, None, None, k, v, nkv * hd, nkv * hd, 1, n)
    for got, x in ((k, K), (v, V)):
        assert np.array_equal(got.numpy(), D.to_f16(D.stands_for(*D.quantise(x, 15))))
    Q = Hn.randn((1, nkv * hd), 3)
    z = up(et, np.zeros((1, nkv * hd), np.float16))
    need = et.mha_kv_workspace(c, 2, 1, 1, nkv)
    et.mha_kv(c, table, 2, up(et, np.array([n - 1], np.int32)), None, up(et, Q), nkv * hd, z, nkv * hd, 1, 1, nkv, 1 / 16, 0, up(et, np.zeros(max(need, 16), np.uint8)), need)
    got = z.numpy()
    Z, stepped, lows, reach = D.attention(host, np.array([[0, 1]], np.int32), [n - 1], [1], Q, 1, nkv, 1 / 16, False)
    assert (np.abs(got - Z) <= allowed(Z, stepped, lows, reach, hd, n)).all()


@pytest.mark.parametrize("max_pages", [50, 300])  # (300: keys are shared out, and the parts joined)
def test_attention_in_a_graph(et, max_pages):
    """A decoding step, written and attended, recorded once and replayed with the position on the device moving on between replays: every
    replay equals the eager calls on a second cache."""
    lib = et.lib()
    nkv, hd, page, B = 2, 64, 16, 3
    nh, width = 4, 128
    first = [30, 700, 15]
    table = tables(3, B, max_pages, B * max_pages)
    host = filled(4, nkv, hd, page, table, first, 1, B * max_pages)
    dev, dev2 = DeviceCache(et, host), DeviceCache(et, host)
    stream = C.c_void_p()
    et.check(lib.et_stream_create(C.byref(stream)))
    dt, ds = up(et, table), up(et, np.array(first, np.int32))
    kv, q = up(et, np.zeros((B, 2 * width), np.float16)), up(et, np.zeros((B, nh * hd), np.float16))
    z, z2 = (up(et, np.zeros((B, nh * hd), np.float16)) for _ in range(2))
    need = et.mha_kv_workspace(dev.c, max_pages, B, 1, nh)
    ws, ws2 = (up(et, np.full(max(need, 16), 0xFF, np.uint8)) for _ in range(2))

    def step(d, out, w, s):
        et.kv_write(d.c, dt, max_pages, ds, None, kv, kv.offset(2 * width), 2 * width, 2 * width, B, 1, s)
        et.mha_kv(d.c, dt, max_pages, ds, None, q, nh * hd, out, nh * hd, B, 1, nh, 0.125, 0, w, need, s)

    step(dev2, z2, ws2, stream)
    et.check(lib.et_stream_sync(stream))
    et.check(lib.et_graph_begin_capture(stream))
    step(dev, z, ws, stream)
    graph = C.c_void_p()
    et.check(lib.et_graph_end_capture(stream, C.byref(graph)))
    for rep in range(5):
        x, y = Hn.randn((B, 2 * width), 50 + rep), Hn.randn((B, nh * hd), 90 + rep)
        at = np.array(first, np.int32) + rep
        for buf, a in ((kv, x), (q, y), (ds, at)):
            et.check(lib.et_memcpy_h2d(buf.ptr, a.ctypes.data, a.nbytes))
        et.check(lib.et_graph_launch(graph, stream))
        step(dev2, z2, ws2, stream)
        et.check(lib.et_stream_sync(stream))
        assert np.array_equal(z.numpy(), z2.numpy()), rep
    for k in dev.bufs:
        assert np.array_equal(dev.bufs[k].numpy().view(np.uint8), dev2.bufs[k].numpy().view(np.uint8))
    et.check(lib.et_graph_destroy(graph))
    et.check(lib.et_stream_destroy(stream))


def test_attention_on_two_streams_at_once(et):
    """Two batches over one cache, keys shared out over workgroups, each with its stream and workspace: what each gives alone."""
    lib = et.lib()
    table = tables(2, 2, 300, 600)
    host = filled(4, 2, 64, 16, table, [4600, 900], 7, 600)
    dev, dt, ds = DeviceCache(et, host), up(et, table), up(et, np.array([4599, 899], np.int32))
    Q = [Hn.randn((2, 256), 5), Hn.randn((2, 256), 6)]
    want = [run_attention(et, dev, table, [4599, 899], None, q, 2, 1, 4, 0.125, False) for q in Q]
    need = et.mha_kv_workspace(dev.c, 300, 2, 1, 4)
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
            et.mha_kv(dev.c, dt, 300, ds, None, q[k], 256, z[k].offset(i * 2 * 256 * 2), 256, 2, 1, 4, 0.125, 0, ws[k], need, s)
    for k, s in enumerate(streams):
        et.check(lib.et_stream_sync(s))
        assert (z[k].numpy() == want[k]).all()
        et.check(lib.et_stream_destroy(s))


def test_attention_gives_the_same_bits_again(et):
    """The order of the sums does not change from run to run, nor with what the workspace held."""
    table = tables(2, 2, 100, 200)
    host = filled(4, 2, 64, 16, table, [1500, 900], 7, 200)
    dev = DeviceCache(et, host)
    Q = Hn.randn((2, 256), 5)
    a = [run_attention(et, dev, table, [1499, 899], None, Q, 2, 1, 4, 0.125, False) for _ in range(3)]
    assert np.array_equal(a[0], a[1]) and np.array_equal(a[0], a[2])
