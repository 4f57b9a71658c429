"""How near et_mha_kv_f16 is to binary64 by the 2-norm, in every kernel that it may run: the roundings of single weights, which a
bound for each value has to grant one by one, show here where they add up."""
import math

import numpy as np
import pytest

from oracle import decode as D
from tests.test_gpu_kv_cache import DeviceCache, run_attention, tables

pytestmark = pytest.mark.gpu

# A result is rounded to binary16 once: off by at most half a step, 2^-11 of it at the lower end of a binade and less above, evenly
# spread, which is 2^-11 / sqrt(3) = 2.82e-4 of the 2-norm at most.  The rest is for what is kept in more bits: weights in two binary16 numbers (2^-22; values that
# cancel in a sum of 5000 make 3e-5 of that if all of them err to one side), binary32 sums and scores.
NEAR = 3e-4

# (hd, key/value heads, query heads to each, rows, lengths): a key a lane (1, 2 and 4 rows), blocks of 16 / groups, of 16, of 8 over pairs of groups; keys of one
# workgroup and keys shared out.
FORMS = [(32, 4, 1, 1, [300, 290]), (64, 4, 1, 1, [300, 290]), (96, 4, 1, 1, [300, 290]), (128, 4, 1, 1, [300, 290]), (64, 4, 2, 1, [300, 290]), (32, 4, 4, 1, [300, 290]),
         (64, 4, 4, 1, [300, 290]), (128, 2, 4, 1, [300, 290]), (160, 2, 4, 1, [300, 290]), (256, 2, 2, 1, [300, 290]), (64, 2, 5, 2, [300, 290]), (96, 2, 16, 1, [300, 290]),
         (128, 2, 3, 4, [300, 290]), (192, 2, 8, 1, [300, 290]), (224, 2, 5, 1, [300, 290]), (256, 2, 8, 1, [300, 290]), (128, 2, 8, 1, [2100, 700]), (64, 2, 1, 1, [5000, 4000]),
         (128, 1, 4, 1, [5000]), (128, 1, 8, 1, [5000]), (128, 1, 16, 1, [5000])]
# without the longest ones but for the last, where there are many cases of each
FEWER = [f for f in FORMS if max(f[4]) < 4000] + FORMS[-1:]


def rows_of(form, seed, values=lambda r, tokens, width: r.standard_normal((tokens, width)) * 0.5):
    """Keys, values and queries of a form, and where its rows stand."""
    hd, nkv, per, n, lengths = form
    r = np.random.default_rng(seed)
    tokens, width = len(lengths) * max(lengths), nkv * hd
    K = (r.standard_normal((tokens, width)) + 1.5 * r.standard_normal(width)).astype(np.float16)
    V = values(r, tokens, width).astype(np.float16)
    Q = r.standard_normal((len(lengths) * n, nkv * per * hd))
    return K, V, Q, [l - n for l in lengths], [n] * len(lengths)


def attended(et, bits, form, seed, qscale=1.0, **kw):
    """(result, the same in binary64), [rows][heads][hd]."""
    hd, nkv, per, n, lengths = form
    K, V, Q, starts, counts = rows_of(form, seed, **kw)
    Q = (Q * qscale).astype(np.float16)
    B, page = len(lengths), 64
    max_pages = -(-max(lengths) // page)
    table = tables(seed, B, max_pages, B * max_pages)
    host = D.Cache(bits, nkv, hd, page, B * max_pages, fill=0xFF)
    host.write(table, [0] * B, lengths, K, V, max(lengths))
    nh = nkv * per
    got = run_attention(et, DeviceCache(et, host), table, starts, counts, Q, B, n, nh, 1 / math.sqrt(hd), True)
    Z = D.attention(host, table, starts, counts, Q, n, nh, 1 / math.sqrt(hd), True)[0]
    return got.astype(np.float64).reshape(-1, nh, hd), Z.reshape(-1, nh, hd)


def off(got, Z):
    """The 2-norm of the error over that of the result, by channel group."""
    by_group = lambda a: a.reshape(-1, a.shape[-1] // 32, 32).transpose(1, 0, 2).reshape(a.shape[-1] // 32, -1)  # noqa: E731
    return np.linalg.norm(by_group(got - Z), axis=1) / np.linalg.norm(by_group(Z), axis=1)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("qscale", [1.0, 2.0 ** -13])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_attention_is_as_near_as_its_result_is_rounded(et, bits, form, qscale):
    """With even probabilities (queries of 2^-13) equal weights are rounded alike and add up: with one binary16 number a weight this is 4e-4 to 9e-4
    (tests/test_decode_precision.py)."""
    got, Z = attended(et, bits, form, 11, qscale)
    e = np.linalg.norm(got - Z) / np.linalg.norm(Z)
    assert e <= NEAR, e


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("qscale", [1.0, 2.0 ** -13])
@pytest.mark.parametrize("every", [2, 4, 7])
@pytest.mark.parametrize("form", FEWER, ids=str)
def test_values_of_single_tokens_far_larger(et, bits, form, every, qscale):
    """Tokens of ordinary values beside tokens whose values are 256 times as large, at any place of four: weights are kept in range by the largest scale of all."""
    got, Z = attended(et, bits, form, 17, qscale, values=lambda r, tokens, width: r.standard_normal((tokens, width)) * np.where(np.arange(tokens) % every == every - 1, 128.0, 0.5)[:, None])
    e = np.linalg.norm(got - Z) / np.linalg.norm(Z)
    assert e <= NEAR, e


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_a_channel_far_larger_in_queries(et, bits, form):
    """One channel of each group is 200 times the others in the queries and small in the keys, whose codes there are about half of the largest: the other channels' terms are 2^-10 of its own
    and less.  What the products drop, 2^-24 of the largest one's place, is 2^-17 of a step times that query, some 1e-4 of a score."""
    hd, nkv, per, n, lengths = form
    K, V, Q, starts, counts = rows_of(form, 18)
    K[:, 2::32] = (K[:, 2::32] * 0.01).astype(np.float16)
    Q[:, 2::32] *= 200
    Q, nh, B = Q.astype(np.float16), nkv * per, len(lengths)
    max_pages = -(-max(lengths) // 64)
    table = tables(18, B, max_pages, B * max_pages)
    host = D.Cache(bits, nkv, hd, 64, B * max_pages, fill=0xFF)
    host.write(table, [0] * B, lengths, K, V, max(lengths))
    got = run_attention(et, DeviceCache(et, host), table, starts, counts, Q, B, n, nh, 1 / math.sqrt(hd), True)
    Z = D.attention(host, table, starts, counts, Q, n, nh, 1 / math.sqrt(hd), True)[0]
    e = np.linalg.norm(got - Z) / np.linalg.norm(Z)
    assert e <= NEAR, e


def alternate(large, small):
    return lambda r, tokens, width: np.clip(r.standard_normal((tokens, width // 32, 32)) * np.where(np.arange(width // 32) % 2, small, large)[:, None], -65504, 65504).reshape(tokens, width)


def turning(large, small):
    """Groups whose values are large in every other stretch of 150 tokens, each in its turn."""
    def values(r, tokens, width):
        size = np.where((np.arange(tokens)[:, None] // 150 + np.arange(width // 32)) % 2, small, large)
        return np.clip(r.standard_normal((tokens, width // 32, 32)) * size[..., None], -65504, 65504).reshape(tokens, width)
    return values


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("qscale", [1.0, 2.0 ** -13])
@pytest.mark.parametrize("form", [f for f in FEWER if f[0] > 32], ids=str)
@pytest.mark.parametrize("values", [alternate(2.0 ** 13, 2.0 ** -7), alternate(2.0 ** -7, 2.0 ** 13), turning(2.0 ** 13, 2.0 ** -7)], ids=["alternate", "alternate2", "turning"])
def test_groups_of_very_different_size(et, bits, form, qscale, values):
    """Channel groups whose values are 2^20 apart are each as near as if they were alone."""
    got, Z = attended(et, bits, form, 12, qscale, values=values)
    e = off(got, Z)
    assert (e <= NEAR).all(), e


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("qscale", [1.0, 2.0 ** -13])
@pytest.mark.parametrize("form", [f for f in FEWER if f[0] > 32], ids=str)
@pytest.mark.parametrize("values", [alternate(2.0 ** 13, 2.0 ** -9), alternate(2.0 ** -9, 2.0 ** 13), turning(2.0 ** -9, 2.0 ** 13)], ids=["alternate", "alternate2", "turning"])
def test_groups_of_very_different_size_further_apart(et, bits, form, qscale, values):
    """2^22: the small ones' results come to where binary16 has subnormal numbers, each off by up to 2^-25, evenly spread."""
    got, Z = attended(et, bits, form, 15, qscale, values=values)
    by_group = lambda a: np.linalg.norm(a.reshape(-1, a.shape[-1] // 32, 32).transpose(1, 0, 2).reshape(a.shape[-1] // 32, -1), axis=1)  # noqa: E731
    e, lim = by_group(got - Z), NEAR * by_group(Z) + 2.0 ** -25 / math.sqrt(3) * math.sqrt(Z.size / (Z.shape[-1] // 32))
    assert (e <= lim).all(), e / lim


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_values_at_the_end_of_the_range(et, bits, form):
    """A group from -65504 to 65504 gets a scale whose last steps lie beyond: what is read back is the largest number, and so is what attention gives."""
    def values(r, tokens, width):
        return np.tile(np.where(np.arange(width) % 3, 65504.0, -65504.0), (tokens, 1))
    got, Z = attended(et, bits, form, 13, values=values)
    assert np.abs(Z).max() > 65520
    want = np.clip(Z, -65504, 65504)
    assert np.isfinite(got).all() and (np.abs(got - want) <= 2.0 ** -10 * np.abs(want)).all()


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_infinite_queries_make_their_row_not_a_number(et, form, bad):
    """Scores of plus or minus infinity have no softmax, whatever the keys' signs; other rows and heads are what they are without them."""
    hd, nkv, per, n, lengths = form
    K, V, Q, starts, counts = rows_of(form, 14)
    B, nh = len(lengths), nkv * per
    max_pages = -(-max(lengths) // 64)
    table = tables(14, B, max_pages, B * max_pages)
    Q = Q.astype(np.float16)
    host = D.Cache(4, nkv, hd, 64, B * max_pages, fill=0xFF)
    host.write(table, [0] * B, lengths, np.abs(K) + np.float16(1), V, max(lengths))
    dev = DeviceCache(et, host)
    want = run_attention(et, dev, table, starts, counts, Q, B, n, nh, 0.1, True).reshape(-1, nh, hd)
    Q[0, 5] = bad
    got = run_attention(et, dev, table, starts, counts, Q, B, n, nh, 0.1, True).reshape(-1, nh, hd)
    assert np.isnan(got[0, 0]).all()
    got[0, 0] = want[0, 0]
    assert np.array_equal(got, want)


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("bad", [np.inf, -np.inf])
def test_infinite_queries_over_keys_of_one_sign(et, form, bad):
    """Every score is plus infinity, or every score is minus infinity: no key's code is 0 where the query is infinite."""
    hd, nkv, per, n, _ = form
    form = (hd, nkv, per, n, [5, 4])
    K, V, Q, starts, counts = rows_of(form, 16)
    nh = nkv * per
    K = np.abs(K) + np.float16(1)
    K[:, 5::hd] = 12
    table = np.array([[1], [0]], np.int32)
    host = D.Cache(4, nkv, hd, 64, 2, fill=0xFF)
    host.write(table, [0, 0], [5, 4], K, V, 5)
    Q = Q.astype(np.float16)
    Q[0, 5] = bad
    got = run_attention(et, DeviceCache(et, host), table, starts, counts, Q, 2, n, nh, 0.1, True).reshape(-1, nh, hd)
    assert np.isnan(got[0, 0]).all() and np.isnan(got).sum() == hd


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd,per,n", [(64, 1, 2), (64, 3, 5), (128, 3, 4), (256, 2, 4)])
def test_not_a_number_of_a_later_token_beside_groups_of_very_different_size(et, bits, hd, per, n):
    """What the rows in front of a token that is NaN give, which do not see it, is the same to the bit whatever it holds; a page without a place in between.  (Against binary64: a result to half a
    step, 2^-11, its group's largest as much again for what cancels, each four times over.)"""
    nkv, lengths = 2, [330, 70]
    r = np.random.default_rng(19)
    K = r.standard_normal((2 * 330, nkv * hd)).astype(np.float16)
    V = alternate(2.0 ** 13, 2.0 ** -9)(r, 2 * 330, nkv * hd).astype(np.float16)
    table = tables(19, 2, 6, 12)
    table[0, 2] = -1
    host = D.Cache(bits, nkv, hd, 64, 12, fill=0xFF)
    host.write(table, [0, 0], lengths, K, V, 330)
    starts = [l - n for l in lengths]
    Q = r.standard_normal((2 * n, nkv * per * hd)).astype(np.float16)
    got = run_attention(et, DeviceCache(et, host), table, starts, None, Q, 2, n, nkv * per, 1 / math.sqrt(hd), True)
    Z = D.attention(host, table, starts, [n, n], Q, n, nkv * per, 1 / math.sqrt(hd), True)[0]
    assert (np.abs(got - Z) <= 2.0 ** -9 * np.abs(Z) + 2.0 ** -9 * np.abs(Z).reshape(2 * n, -1, 32).max(-1).repeat(32, -1)).all()
    row = np.full((2, nkv * hd), np.nan, np.float16)
    host.write(table, [l - 1 for l in lengths], [1, 1], row, row, 1)
    again = run_attention(et, DeviceCache(et, host), table, starts, None, Q, 2, n, nkv * per, 1 / math.sqrt(hd), True)
    last = np.arange(2 * n) % n == n - 1
    assert np.array_equal(got[~last], again[~last]) and np.isnan(again[last]).all()
