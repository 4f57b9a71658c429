"""4-bit weights: made of a dense weight bit for bit as the format says, expanded again, and multiplied, against binary64."""
import ctypes as C

import numpy as np
import pytest

from oracle import decode as D
from tests import harness as Hn
from tests.harness import up
from tests.test_gpu_kv_cache import hard_values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("out,n", [(16, 1), (48, 3), (272, 10)])
def test_quantise_and_expand(et, group, out, n):
    n_in = n * group
    W = hard_values((out, n_in), 5)
    codes = up(et, np.full((out, n_in // 2), 0xA5, np.uint8))
    scales = up(et, np.full((n, out, 2), np.nan, np.float16))
    et.dense_to_w4(up(et, W), codes, scales, n_in, out, group)
    want_c, want_s = D.w4_pack(W, group)
    assert np.array_equal(codes.numpy(), want_c)
    assert np.array_equal(scales.numpy(), want_s)
    back = up(et, np.zeros((out, n_in), np.float16))
    et.w4_to_dense(codes, scales, back, n_in, out, group)
    assert np.array_equal(back.numpy(), D.to_f16(D.w4_dense(want_c, want_s, group)))


def test_not_a_number_stays_in_its_group(et):
    W = Hn.randn((32, 128), 1)
    W[3, 70], W[9, 0] = np.nan, np.inf
    codes, scales, back = up(et, np.zeros((32, 64), np.uint8)), up(et, np.zeros((2, 32, 2), np.float16)), up(et, np.zeros((32, 128), np.float16))
    et.dense_to_w4(up(et, W), codes, scales, 128, 32, 64)
    et.w4_to_dense(codes, scales, back, 128, 32, 64)
    bad = np.isnan(back.numpy())
    assert bad[3, 64:].all() and bad[9, :64].all() and bad.sum() == 128


def reference(W, x, bias, act):
    """(result, what it may be off by but for the last rounding): every product and sum in binary32 is one of at most `in` + 64 roundings of
    2^-24 in sums of magnitude sum |x| (|scale| code + |low|); GELU's slope is below 1.13, its own exp2 and reciprocal are good to 2^-20."""
    w, size = W
    y = x @ w.T + bias
    off = (x.shape[1] + 64) * 2.0 ** -24 * (np.abs(x) @ size.T + np.abs(bias))
    if act == 1:
        y = np.maximum(y, 0)
    elif act == 2:
        u = y * (0.035677408136 * y * y + 0.7978845608028654)
        y, off = y * (0.5 + 0.5 * np.tanh(u)), 1.13 * off + 2.0 ** -19 * np.abs(y)
    return y, off


def weight(codes, scales, group):
    """Its values, and |scale| code + |low|."""
    return D.w4_dense(codes, scales, group), D.w4_dense(codes, np.abs(scales), group)


def run(et, codes, scales, group, bias, x, act, f32, stream=None):
    T, n_in = x.shape
    out = codes.shape[0]
    y = up(et, np.full((T + 1, out), -77, np.float32 if f32 else np.float16))
    et.linear_w4(up(et, codes), up(et, scales), group, None if bias is None else up(et, bias), up(et, x), None if f32 else y, y if f32 else None, T, n_in, out, act, stream)
    got = y.numpy()
    assert (got[T] == -77).all()
    return got[:T].astype(np.float64)


def check(et, T, n_in, out, group, act, f32, with_bias=True, xs=1.0, seed=0):
    r = np.random.default_rng(seed + T)
    codes, scales = D.w4_pack((r.standard_normal((out, n_in)) * 0.05 + 0.02).astype(np.float16), group)
    x = (r.standard_normal((T, n_in)) * xs).astype(np.float16)
    bias = r.standard_normal(out).astype(np.float16) if with_bias else None
    got = run(et, codes, scales, group, bias, x, act, f32)
    y, off = reference(weight(codes, scales, group), x.astype(np.float64), bias.astype(np.float64) if with_bias else np.zeros(out), act)
    lim = off + (2.0 ** -24 if f32 else 2.0 ** -11) * np.abs(y) + (0 if f32 else 2.0 ** -25)
    assert (np.abs(got - y) <= lim).all(), np.max(np.abs(got - y) / lim)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 31, 32, 33, 47, 48, 64, 65, 100, 130])
def test_rows(et, T, group):
    check(et, T, 384, 80, group, 0, T % 2 == 1, seed=group)


@pytest.mark.parametrize("n_in,out,group", [(32, 16, 32), (64, 16, 64), (128, 16, 128), (160, 48, 32), (192, 32, 64), (800, 208, 32), (1024, 256, 64), (2176, 64, 128),
                                            (4096, 1040, 128), (16384, 32, 32), (96, 4096, 32)])
@pytest.mark.parametrize("T", [1, 6, 20, 70])
def test_sizes(et, T, n_in, out, group):
    check(et, T, n_in, out, group, T % 3, False, with_bias=out != 64)


@pytest.mark.parametrize("T,out", [(1, 16400), (4, 8208), (4, 16416), (16, 8208), (16, 16416), (32, 8192), (45, 8208), (64, 4080), (64, 8224), (600, 1072), (70001, 16)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_many_output_features_or_rows(et, T, out, group):
    """Waves that take several blocks of 16 output features, the last of them none; more rows than a grid's second dimension has numbers."""
    check(et, T, 384, out, group, 0, False)


@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("with_bias", [False, True])
def test_epilogues(et, act, f32, with_bias):
    for T in (1, 13, 40):
        check(et, T, 256, 96, 64, act, f32, with_bias)


@pytest.mark.parametrize("xs", [2.0 ** -14, 2.0 ** -20, 1000.0])
def test_inputs_of_other_sizes(et, xs):
    """Activations among the subnormal numbers of binary16 keep their bits; large ones do not overflow before the scale is applied."""
    check(et, 3, 256, 48, 32, 0, True, with_bias=False, xs=xs)
    check(et, 20, 256, 48, 128, 0, True, with_bias=False, xs=xs)


def test_infinity_and_nan_of_a_row_stay_in_it(et):
    codes, scales = D.w4_pack(Hn.randn((32, 128), 3, 0.1), 32)
    for T in (4, 20):
        x = Hn.randn((T, 128), 4)
        x[1, 5], x[3, 77] = np.nan, np.inf
        got = run(et, codes, scales, 32, None, x, 0, True)
        rows = np.ones(T, bool)
        rows[[1, 3]] = False
        assert np.isnan(got[1]).all() and not np.isfinite(got[3]).any() and np.isfinite(got[rows]).all()


def test_weight_beyond_32_bits_of_bytes(et):
    """Codes of more than 4 GiB: the last output features of a weight of zeros but for those."""
    n_in, out, group = 65536, 131072 + 32, 128
    codes, scales = et.DeviceBuffer(n_in // 2 * out), et.DeviceBuffer(n_in // group * out * 4)
    tail_c, tail_s = D.w4_pack(Hn.randn((16, n_in), 1, 0.01), group)
    et.check(et.lib().et_memcpy_h2d(codes.offset((out - 16) * (n_in // 2)), tail_c.ctypes.data, tail_c.nbytes))
    for g in range(n_in // group):
        row = np.ascontiguousarray(tail_s[g])
        et.check(et.lib().et_memcpy_h2d(scales.offset((g * out + out - 16) * 4), row.ctypes.data, row.nbytes))
    x = Hn.randn((1, n_in), 2)
    y = et.DeviceBuffer(out * 4)
    et.linear_w4(codes, scales, group, None, up(et, x), None, y, 1, n_in, out)
    got = y.numpy(np.float32, (out,)).astype(np.float64)
    assert (got[:-16] == 0).all()
    want, off = reference(weight(tail_c, tail_s, group), x.astype(np.float64), np.zeros(16), 0)
    assert (np.abs(got[-16:] - want[0]) <= off[0] + 2.0 ** -24 * np.abs(want[0])).all()


def test_graph_replays(et):
    lib = et.lib()
    codes, scales = (up(et, a) for a in D.w4_pack(Hn.randn((512, 1024), 3, 0.05), 64))
    x, y, want = up(et, Hn.randn((2, 1024), 4)), up(et, np.zeros((2, 512), np.float16)), up(et, np.zeros((2, 512), np.float16))
    stream, graph = C.c_void_p(), C.c_void_p()
    et.check(lib.et_stream_create(C.byref(stream)))
    et.linear_w4(codes, scales, 64, None, x, want, None, 2, 1024, 512, 0, stream)
    et.check(lib.et_stream_sync(stream))
    et.check(lib.et_graph_begin_capture(stream))
    et.linear_w4(codes, scales, 64, None, x, y, None, 2, 1024, 512, 0, stream)
    et.check(lib.et_graph_end_capture(stream, C.byref(graph)))
    for rep in range(3):
        new = Hn.randn((2, 1024), 10 + rep)
        et.check(lib.et_memcpy_h2d(x.ptr, new.ctypes.data, new.nbytes))
        et.check(lib.et_graph_launch(graph, stream))
        et.linear_w4(codes, scales, 64, None, x, want, None, 2, 1024, 512, 0, stream)
        et.check(lib.et_stream_sync(stream))
        assert np.array_equal(y.numpy(), want.numpy())
    et.check(lib.et_graph_destroy(graph))
    et.check(lib.et_stream_destroy(stream))
