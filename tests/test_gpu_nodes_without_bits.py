"""Trees under a window whose nodes have any bits, none among them: a node without bits has depth 0, and sees no more than the first node, wherever its window begins in a tile or a page."""
import numpy as np
import pytest

from oracle import sight as S
from tests.test_gpu_sight import check_tree


def words_of(B, n):
    """Any bits; none in the first row, in every fifth, and in all rows of some sequences."""
    words = np.random.default_rng(n).integers(0, 2 ** 32, (B, n, (n + 31) // 32), dtype=np.uint32)
    words[:, ::5], words[::7] = 0, 0
    return words


def test_the_oracle_sees_no_page_that_was_given_back():
    """What a row sees before the call's rows is in pages that et_kv_tables calls needed."""
    page, M, n = 16, 14, 4
    for start in range(64, 192):
        for window in (4, 50):
            table = S.tables(np.full((1, M), -1, np.int32), page, M, [start], [n], None, n, window, 0, np.arange(M, dtype=np.int32), np.array([0, M, 0], np.int32))[0]
            for words in (words_of(1, n), np.full((1, n, 1), 2 ** 32 - 1, np.uint32)):
                sees = S.tree_sight([start], [n], n, words, window, 0)
                pos = np.arange(start)
                for i in range(n):
                    assert (table[0, pos[sees(0, i, pos)] // page] >= 0).all(), (start, window, i)


# (query heads over each key/value head, hd, nodes, batches alike): a key a lane, blocks of 16 / groups, blocks of 16, 256 and 64 rows a workgroup
@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("per,hd,n,copies", [(1, 64, 1, 1), (4, 128, 1, 1), (1, 64, 6, 1), (3, 96, 2, 1), (1, 64, 40, 1), (8, 256, 2, 1), (4, 128, 40, 4), (4, 128, 12, 12), (1, 64, 130, 8), (4, 32, 40, 8)])
def test_windows_that_begin_anywhere(et, page, per, hd, n, copies):
    window = max(50, n)
    check_tree(et, 4, 1, per, hd, page, [window + 64 + i for i in range(64)], [n] * 64, n, window, 0, seed=n, words=words_of(64, n), copies=copies)
