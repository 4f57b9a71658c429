"""What the 2-norm that attention over a quantised cache is held to (tests/test_gpu_kv_precision.py) tells apart: the sums in numpy, weights rounded to one binary16 number and to two."""
import numpy as np
import pytest

from oracle import decode as D
from tests.test_gpu_kv_precision import NEAR


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("keys", [290, 700, 5000])
def test_a_weight_in_one_binary16_number_shows(bits, keys):
    """Even probabilities p; results are rounded to binary16 as the kernels round theirs."""
    r = np.random.default_rng(keys)
    codes, scale, low = D.quantise((r.standard_normal((keys, 512)) * 0.5).astype(np.float16), 2 ** bits - 1)
    y = r.standard_normal((keys, 1)) * 1e-3
    p = np.exp2(y - y.max() + 11.37)  # (the largest weight's place, as a running maximum leaves it)
    weight = p * np.repeat(scale.astype(np.float64), 32, 1)
    lows = p * np.repeat(low.astype(np.float64), 32, 1)
    Z = (weight * codes + lows).sum(0) / p.sum()
    one = weight.astype(np.float32).astype(np.float16).astype(np.float64)
    two = one + (weight - one).astype(np.float16).astype(np.float64)

    def off(w):
        return np.linalg.norm(((w * codes + lows).sum(0) / p.sum()).astype(np.float16).astype(np.float64) - Z) / np.linalg.norm(Z)

    assert off(two) <= NEAR < off(one)
