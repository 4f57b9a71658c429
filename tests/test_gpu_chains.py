"""A tree that is a chain, and a window that hides nothing, are causal attention over all keys (et_mha_kv_f16): the kernels with sight against those without."""
import numpy as np
import pytest

from oracle import decode as D
from oracle import sight as S
from tests import harness as Hn
from tests.test_gpu_kv_cache import DeviceCache, filled, run_attention, tables
from tests.test_gpu_sight import run_tree, run_window

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("per,hd,n", [(1, 64, 1), (2, 32, 1), (4, 128, 1), (8, 256, 1), (1, 64, 2), (3, 96, 5), (4, 128, 2), (4, 128, 5), (2, 160, 12), (1, 64, 30)])
def test_chains_are_causal_attention(et, bits, per, hd, n):
    """Up to 32 rows a key/value head the sums are the same in the same order: the same bits."""
    B, lengths, nkv = 3, [75, 40, 0], 2
    table = tables(1, B, 7, 21)
    host = filled(bits, nkv, hd, 16, table, [l + n for l in lengths], 4, 21)
    dev, Q, counts = DeviceCache(et, host), Hn.randn((B * n, nkv * per * hd), 5), [n, max(1, n - 1), n]
    words = S.seen_words(np.tile(np.arange(n, dtype=np.int32) - 1, (B, 1)), counts, n)
    want = run_attention(et, dev, table, lengths, counts, Q, B, n, nkv * per, 0.1, True)
    assert np.array_equal(run_tree(et, dev, table, lengths, counts, words, Q, B, n, nkv * per, 0, 0, 0.1), want)
    assert np.array_equal(run_window(et, dev, table, lengths, counts, Q, B, n, nkv * per, 1 << 20, 0, 0.1, True), want)
    Z = D.attention(host, table, lengths, counts, Q, n, nkv * per, 0.1, True)[0]
    there = ~np.isnan(Z[:, 0])
    assert np.abs(want[there] - Z[there]).max() <= 2.0 ** -8 * np.abs(Z[there]).max()
