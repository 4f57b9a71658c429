"""Attention over a window or a tree with many rows a key/value head, by the kernels that turn codes into numbers before they multiply them, where numbers are hard to keep: values of a
few of binary16's smallest steps, and results of which nearly everything cancels, so that what numbers lose is not behind the result's own rounding.  Against binary64."""
import math

import numpy as np
import pytest

from oracle import decode as D
from oracle import sight as S
from tests.test_gpu_kv_cache import DeviceCache
from tests.test_gpu_kv_precision import NEAR, alternate, off, turning
from tests.test_gpu_sight import distance, first, large_channel, near, run_window

pytestmark = pytest.mark.gpu

# (hd, query heads, rows, batches alike or apart): one key/value head, eight waves a workgroup, and two of them a block of 64 rows
MANY = [(32, 4, 40, 320), (64, 1, 130, 320), (96, 3, 70, 320), (128, 8, 20, 220), (128, 4, 16, 480)]
PAGE, PAGES = 64, 5


def attended(et, bits, form, K, V, Q, scale, pages=PAGES):
    """Rows that all see every token, K and V [sequences][tokens][hd], Q [sequences][rows][heads * hd]; (result, then what S.attention gives), a table of so many pages for each sequence.
    One sequence stands for as many as the form has."""
    hd, nh, n, copies = form
    B, tokens = K.shape[:2]
    table = np.full((B, pages), -1, np.int32)
    used = -(-tokens // PAGE)
    table[:, :used] = np.arange(B * used).reshape(B, used)
    host = D.Cache(bits, 1, hd, PAGE, B * used, fill=0xFF)
    host.write(table, [0] * B, [tokens] * B, K.reshape(-1, hd), V.reshape(-1, hd), tokens)
    starts, counts, times = [tokens - n] * B, [n] * B, copies // B
    got = run_window(et, DeviceCache(et, host), np.tile(table, (times, 1)), starts * times, counts * times, np.tile(Q.reshape(B * n, -1), (times, 1)), B * times, n, nh, 1 << 20, 0, scale, False)
    return first(times, got), S.attention(host, table, starts, counts, Q.reshape(B * n, -1), n, nh, scale, S.window_sight(starts, counts, n, 1 << 20, 0, False))


def small(r, *shape):
    """Multiples of 2^-24 up to 40 of them, groups that are all 1, 3 and 17, and numbers about 2^-14 and 2^-13."""
    x = r.integers(1, 41, shape)
    kind = r.integers(0, 8, shape[:-1] + (shape[-1] // 32,)).repeat(32, -1)
    for k, whole in ((0, 1), (1, 3), (2, 17)):
        x = np.where(kind == k, whole, x)
    x = np.where(kind == 3, x + 1024, np.where(kind == 4, x + 2047, x))
    return (x * 2.0 ** -24).astype(np.float16)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("form", MANY, ids=str)
def test_values_of_the_smallest_steps(et, bits, form):
    hd, nh, n, _ = form
    r = np.random.default_rng(hd)
    K, Q = r.standard_normal((1, 300, hd)).astype(np.float16), r.standard_normal((1, n, nh * hd)).astype(np.float16)
    got, want = attended(et, bits, form, K, small(r, 1, 300, hd), Q, 1 / math.sqrt(hd))
    near(got, *want, hd, 300, nh * n)
    # one number alone comes out as it is
    for whole in (1, 3, 5, 17, 1025, 2047):
        got, _ = attended(et, bits, form, K, np.full((1, 300, hd), whole * 2.0 ** -24, np.float16), Q, 1 / math.sqrt(hd))
        assert (got == np.float16(whole * 2.0 ** -24)).all(), (whole, np.unique(got.astype(np.float64) * 2.0 ** 24))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("form", MANY, ids=str)
def test_keys_of_the_smallest_steps(et, bits, form):
    """Against queries near the largest numbers, so that a step of a key is some tenths of a score."""
    hd, nh, n, _ = form
    r = np.random.default_rng(hd)
    K = (r.integers(1, 41, (1, 300, 1)) + r.integers(0, 2, (1, 300, hd))).astype(np.float64) * 2.0 ** -24
    V, Q = r.standard_normal((1, 300, hd)).astype(np.float16), (5e4 + 1e4 * r.random((1, n, nh * hd))).astype(np.float16)
    got, want = attended(et, bits, form, K.astype(np.float16), V, Q, 64 / hd)
    near(got, *want, hd, 300, nh * n)


def kept(got, want, hd, keys):
    """Held to what a key's and a value's number in two binary16 numbers leaves (the first cut off: 2^-10 of it, the second rounded: 2^-11 of that), as a weight's two do (2^-22), the product of
    second parts that is left out (2^-10 times 2^-11), and binary32: scores off by d, from 2^-21 of their terms, hd + 16 roundings of 2^-24 in sums of magnitude `reach` and
    2^-20 for exp2, move every p by 2 d; a sum over the keys has keys + 16 roundings.  The result is rounded once: 2^-11, or 2^-25 where it is subnormal."""
    Z, stepped, lows, reach = want
    d = ((hd + 16) * 2.0 ** -24 + 2.0 ** -21) * reach + 2.0 ** -20
    lim = 2.0 ** -11 * np.abs(Z) + 2.0 ** -25 + (np.expm1(2 * d) + (keys + 16) * 2.0 ** -24 + 3 * 2.0 ** -21) * (stepped + lows)
    off = np.abs(got.astype(np.float64) - Z)
    assert (off <= lim).all(), np.nanmax(off / lim)


def groups(r, bits, B, hd):
    """For each sequence a row whose channels, but for two of every 32, are one number, a step between 1 and 2 that takes more than binary16's bits."""
    x = np.empty((B, 1, hd))
    for b in range(B):
        low, high = np.float64(np.float16(1 + 0.4 * r.random())), np.float64(np.float16(1.5 + 0.49 * r.random()))
        x[b] = low + (high - low) * r.integers(1, 2 ** bits - 1) / (2 ** bits - 1)
        x[b, 0, 0::32], x[b, 0, 1::32] = low, high
    return x.astype(np.float16)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("form", MANY, ids=str)
def test_values_that_nearly_cancel(et, bits, form):
    """Every other token has the opposite values of the others, but for what its codes make of them: what a value loses stays."""
    hd, nh, n, copies = form
    r, B, tokens = np.random.default_rng(hd), copies // 2, 32
    V = np.repeat((1 + r.random((B, 1, hd))).astype(np.float16), tokens, 1)
    V[:, 1::2] *= -1
    got, want = attended(et, bits, form, np.zeros((B, tokens, hd), np.float16), V, r.standard_normal((B, n, nh * hd)).astype(np.float16), 0.1)
    kept(got, want, hd, tokens)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("form", MANY, ids=str)
def test_weights_that_nearly_cancel(et, bits, form):
    """One token is weighed more and has no values; four times 1.249 and five times -1 are what the others have, all with one weight, which takes more than binary16's bits."""
    hd, nh, n, copies = form
    r, B = np.random.default_rng(hd + 1), copies // 2
    K, V = np.zeros((B, 10, hd)), np.zeros((B, 10, hd))
    K[:, 0] = 1
    V[:, 1:5], V[:, 5:] = 1.249, -1
    Q = np.repeat((0.5 + r.random((B, 1, 1))), nh * hd, 2).repeat(n, 1)
    got, want = attended(et, bits, form, K.astype(np.float16), V.astype(np.float16), Q.astype(np.float16), 2 / hd)
    kept(got, want, hd, 10)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("form", MANY, ids=str)
def test_scores_that_nearly_agree(et, bits, form):
    """Two kinds of tokens with scores of about 10 to 20 and values of 1 and -1: the result is half of the difference of their scores."""
    hd, nh, n, copies = form
    r, B, tokens = np.random.default_rng(hd + 2), copies // 2, 32
    K = np.repeat(groups(r, bits, B, hd), tokens, 1)
    K[:, 1::2] = groups(r, bits, B, hd)
    Q = np.repeat((1 + 0.25 * r.random((B, 1, 1))), nh * hd, 2).repeat(n, 1)
    V = np.ones((B, tokens, hd))
    V[:, 1::2] = -1
    got, want = attended(et, bits, form, K, V.astype(np.float16), Q.astype(np.float16), 8 / hd)
    kept(got, want, hd, tokens)


# keys shared out over workgroups, eight waves of each and two pairs of two, and joined: (form, pages of the table, tokens)
SHARED = [((128, 1, 70, 16), 32, 2000), ((128, 2, 128, 8), 64, 1500), ((64, 1, 130, 16), 94, 2000), ((128, 4, 10, 32), 63, 2000), ((128, 1, 64, 1), 2000, 700)]


def spread(et, bits, form, pages, tokens, seed, values=lambda r, tokens, width: r.standard_normal((tokens, width)) * 0.5, qscale=1.0, keys=None):
    """(result, the same in binary64), [rows][heads][hd]."""
    hd, nh, n, _ = form
    r = np.random.default_rng(seed)
    K = (r.standard_normal((tokens, hd)) + 1.5 * r.standard_normal(hd)).astype(np.float16)
    V, Q = values(r, tokens, hd).astype(np.float16), r.standard_normal((n, nh * hd)) * qscale
    if keys:
        K, Q = keys(K, Q)
    got, want = attended(et, bits, form, K[None], V[None], Q.astype(np.float16)[None], 1 / math.sqrt(hd), pages)
    return got.astype(np.float64).reshape(n, nh, hd), want[0].reshape(n, nh, hd)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("form,pages,tokens", SHARED, ids=str)
def test_shared_out(et, bits, form, pages, tokens):
    """Ordinary values, single tokens whose values are far larger, a channel far larger in queries, even probabilities."""
    far = lambda every: lambda r, t, width: r.standard_normal((t, width)) * np.where(np.arange(t) % every == every - 1, 128.0, 0.5)[:, None]  # noqa: E731
    for more in ({}, dict(values=far(2)), dict(values=far(7)), dict(keys=large_channel), dict(qscale=2.0 ** -13)):
        assert distance(*spread(et, bits, form, pages, tokens, 17, **more)) <= NEAR, more


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("form,pages,tokens", SHARED, ids=str)
def test_shared_out_groups_of_very_different_size(et, bits, form, pages, tokens):
    for qscale in (1.0, 2.0 ** -13):
        for values in (alternate(2.0 ** 13, 2.0 ** -7), turning(2.0 ** 13, 2.0 ** -7)):
            assert (off(*spread(et, bits, form, pages, tokens, 21, values, qscale)) <= NEAR).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("form,pages,tokens", SHARED, ids=str)
def test_shared_out_at_the_end_of_the_range(et, bits, form, pages, tokens):
    got, Z = spread(et, bits, form, pages, tokens, 13, lambda r, t, width: np.tile(np.where(np.arange(width) % 3, 65504.0, -65504.0), (t, 1)), 2.0 ** -17,
                    lambda K, Q: (np.where(K > 0, np.float16(65504), np.float16(-65504)), Q))
    want = np.clip(Z, -65504, 65504)
    assert np.isfinite(got).all() and (np.abs(got - want) <= 2.0 ** -10 * np.abs(want)).all()


@pytest.mark.parametrize("form,pages,tokens", SHARED, ids=str)
def test_shared_out_infinite_queries_make_their_row_not_a_number(et, form, pages, tokens):
    want, _ = spread(et, 4, form, pages, tokens, 14, keys=lambda K, Q: (np.abs(K) + np.float16(1), Q))
    for bad in (np.inf, -np.inf, np.nan):
        def put(K, Q):
            Q[0, 5] = bad
            return np.abs(K) + np.float16(1), Q
        with np.errstate(invalid="ignore"):
            got, _ = spread(et, 4, form, pages, tokens, 14, keys=put)
        assert np.isnan(got[0, 0]).all()
        got[0, 0] = want[0, 0]
        assert np.array_equal(got, want)
