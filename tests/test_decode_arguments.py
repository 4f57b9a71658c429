"""What et_kv_*, et_mha_kv_* and et_*w4* refuse, before anything is launched, and the formats' own bounds."""
import ctypes as C
import math

import numpy as np
import pytest

from oracle import decode as D

P = 1 << 20  # an address that nothing reads: aligned


def cache(et, **kw):
    args = dict(k_codes=P, k_scales=P, v_codes=P, v_scales=P, bits=4, nkv=2, hd=64, page=16, npages=4)
    args.update(kw)
    return et.KvCache(*args.values())


BAD_CACHE = [(dict(k_codes=None), -1), (dict(v_scales=None), -1), (dict(bits=2), -1), (dict(bits=16), -1), (dict(nkv=0), -1), (dict(npages=0), -1), (dict(page=0), -1),
             (dict(hd=0), -1), (dict(hd=48), -2), (dict(hd=288), -2), (dict(page=24), -2), (dict(k_codes=P + 8), -2), (dict(k_scales=P + 4), -2), (dict(nkv=1 << 20), -2)]


def calls(et, c, table=P, max_pages=4, B=1, n=1, ldk=128, ldq=256, K=P, V=P, Q=P, Z=P, nh=4, flags=0, ws=P, ws_bytes=1 << 30):
    lib = et.lib()
    ref = C.byref(c)
    return {"write": lib.et_kv_write_f16(ref, table, max_pages, None, None, K, V, ldk, ldk, B, n, None),
            "read": lib.et_kv_read_f16(ref, table, max_pages, None, None, K, V, ldk, ldk, B, n, None),
            "mha": lib.et_mha_kv_f16(ref, table, max_pages, None, None, Q, ldq, Z, ldq, B, n, nh, 0.1, flags, ws, ws_bytes, None)}


@pytest.mark.parametrize("bad,status", BAD_CACHE)
def test_caches_that_are_none(et, bad, status):
    c = cache(et, **bad)
    wide = 1 << 30
    assert set(calls(et, c, ldk=wide, ldq=wide, nh=max(1, c.nkv)).values()) == {status}
    n = C.c_size_t()
    assert et.lib().et_mha_kv_workspace(C.byref(c), 4, 1, 1, max(1, c.nkv), C.byref(n)) == status
    assert et.lib().et_last_error().startswith(b"et_mha_kv_workspace:")


def test_other_arguments(et):
    c = cache(et)
    lib = et.lib()
    assert set(calls(et, c, table=None).values()) == {-1}
    assert set(calls(et, c, table=P + 2).values()) == {-2}
    assert set(calls(et, c, max_pages=0).values()) == {-1}
    assert set(calls(et, c, max_pages=1 << 28).values()) == {-2}
    assert set(calls(et, c, B=-1).values()) == {-1}
    assert set(calls(et, c, n=-1).values()) == {-1}
    assert set(calls(et, c, ldk=120, ldq=248).values()) == {-1}
    assert set(calls(et, c, ldk=132, ldq=260).values()) == {-2}
    assert set(calls(et, c, K=P + 8, Q=P + 8).values()) == {-2}
    assert set(calls(et, c, B=1 << 20, n=1 << 30).values()) == {-2}
    assert calls(et, c, K=None, n=0)["write"] == -1
    assert calls(et, c, Q=None, n=0)["mha"] == -1 and calls(et, c, Z=None, n=0)["mha"] == -1
    for bad in (dict(nh=3), dict(nh=0), dict(nh=-2), dict(flags=2)):
        assert calls(et, c, n=0, **bad)["mha"] == -1, bad
    # nothing to do: fine, and nothing is launched
    assert set(calls(et, c, B=0).values()) == {0} and set(calls(et, c, n=0).values()) == {0}
    assert lib.et_kv_read_f16(C.byref(c), P, 4, None, None, None, None, 0, 0, 1, 1, None) == 0
    need = C.c_size_t(7)
    assert lib.et_mha_kv_workspace(C.byref(c), 4, 0, 1, 4, C.byref(need)) == 0 and need.value == 0
    assert lib.et_mha_kv_workspace(None, 4, 1, 1, 4, C.byref(need)) == -1
    assert lib.et_mha_kv_workspace(C.byref(c), 4, 1, 1, 4, None) == -1
    assert lib.et_kv_write_f16(None, P, 4, None, None, P, P, 128, 128, 1, 1, None) == -1


def test_the_largest_sizes(et):
    """Positions, threads of a launch and scores that 32 bits would not hold."""
    c = cache(et, page=1 << 20, npages=1, nkv=1, hd=32)
    n = C.c_size_t()
    for pages, status in ((2047, 0), (2048, -2)):
        assert et.lib().et_mha_kv_workspace(C.byref(c), pages, 1, 1, 1, C.byref(n)) == status, pages
    c = cache(et, page=16, npages=1, nkv=1, hd=32)
    for pages, status in ((134217720, 0), (134217721, -2)):  # 2^31 - 128
        assert et.lib().et_mha_kv_workspace(C.byref(c), pages, 1, 1, 1, C.byref(n)) == status, pages
    c = cache(et)
    many = calls(et, c, n=(1 << 29) + 64)  # rows of four groups
    assert many["write"] == many["read"] == -2
    assert linear(et, T=65535 * 32 + 1) == -2 and linear(et, T=0, n_in=(1 << 23) + 32) == -2
    for scale in (math.nan, math.inf, -math.inf, 1.1e15):
        assert et.lib().et_mha_kv_f16(C.byref(c), P, 4, None, None, P, 256, P, 256, 1, 0, 4, scale, 0, P, 1 << 30, None) == -1, scale
    for scale in (1e15, -1e15, 0.0):
        assert et.lib().et_mha_kv_f16(C.byref(c), P, 4, None, None, P, 256, P, 256, 1, 0, 4, scale, 0, P, 1 << 30, None) == 0, scale


def test_workspace_does_not_grow_with_fewer_pages(et):
    """A call with fewer pages than the workspace was made for fits."""
    for nkv, hd, bits, B, n, nh in ((1, 64, 4, 1, 1, 1), (8, 128, 4, 1, 1, 32), (8, 96, 8, 3, 7, 8), (16, 64, 4, 40, 1, 16), (2, 256, 8, 2, 40, 16), (8, 128, 4, 2, 1, 64), (8, 128, 8, 33, 7, 8)):
        c = cache(et, nkv=nkv, hd=hd, bits=bits, npages=1 << 14)
        need = [et.mha_kv_workspace(c, pages, B, n, nh) for pages in range(1, 9000, 37)]
        assert need == sorted(need)


@pytest.mark.parametrize("page", [16, 48, 64])
@pytest.mark.parametrize("nkv,per,B,n", [(8, 8, 4, 1), (1, 1, 1, 7), (2, 5, 3, 1), (3, 3, 2, 2), (4, 7, 63, 1), (8, 4, 4, 1), (2, 9, 1, 1)])
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
def test_workspace_grows_with_every_page(et, hd, nkv, per, B, n, page):
    """Also by one page at a time around the sizes at which another kernel is chosen."""
    for bits in (4, 8):
        c = cache(et, nkv=nkv, hd=hd, bits=bits, page=page, npages=1 << 14)
        need = [et.mha_kv_workspace(c, pages, B, n, nkv * per) for pages in range(1, 6400 // page)]
        assert need == sorted(need), [i + 1 for i in range(len(need) - 1) if need[i] > need[i + 1]]


def test_workspace_is_asked_for(et):
    """One sequence of a million tokens on one head is shared out: what the parts leave needs memory, and a call without it is refused."""
    c = cache(et, nkv=1, npages=1 << 16)
    pages = 1 << 16
    need = et.mha_kv_workspace(c, pages, 1, 1, 1)
    assert need > 0
    for ws, have in ((None, need), (P, need - 1), (P + 8, need)):
        assert calls(et, c, max_pages=pages, nh=1, ws=ws, ws_bytes=have)["mha"] == (-2 if ws == P + 8 else -1), (ws, have)
        assert b"workspace" in et.lib().et_last_error()


def linear(et, codes=P, scales=P, group=32, bias=P, X=P, Y=P, Y32=None, T=1, n_in=64, out=16, act=0):
    return et.lib().et_linear_w4_f16(codes, scales, group, bias, X, Y, Y32, T, n_in, out, act, None)


@pytest.mark.parametrize("bad,status", [(dict(codes=None), -1), (dict(scales=None), -1), (dict(X=None), -1), (dict(Y=None), -1), (dict(Y32=P), -1), (dict(group=16), -1),
                                        (dict(group=96), -1), (dict(n_in=0), -1), (dict(out=0), -1), (dict(T=-1), -1), (dict(act=3), -1), (dict(n_in=48), -2),
                                        (dict(group=128), -2), (dict(out=24), -2), (dict(codes=P + 8), -2), (dict(X=P + 2), -2), (dict(Y=P + 8), -2), (dict(bias=P + 4), -2),
                                        (dict(n_in=1 << 20, out=1 << 20), -2)])
def test_weights_that_are_none(et, bad, status):
    assert linear(et, **bad) == status
    assert linear(et, **{**bad, "T": bad.get("T", 0)}) == status
    assert et.lib().et_last_error().startswith(b"et_linear_w4_f16:")
    if not set(bad) & {"X", "Y", "Y32", "T", "act", "bias"}:
        a = {**dict(codes=P, scales=P, n_in=64, out=16, group=32), **bad}
        assert et.lib().et_dense_to_w4_f16(P, a["codes"], a["scales"], a["n_in"], a["out"], a["group"], None) == status
        assert et.lib().et_w4_to_dense_f16(a["codes"], a["scales"], P, a["n_in"], a["out"], a["group"], None) == status


def test_no_rows(et):
    assert linear(et, T=0) == 0


@pytest.mark.parametrize("levels,group", [(15, 32), (255, 32), (15, 64), (15, 128)])
def test_a_value_is_half_a_step_off_at_most(levels, group):
    r = np.random.default_rng(1)
    x = np.concatenate([r.standard_normal((40, 256)), r.standard_normal((40, 256)) * 2.0 ** -20, r.choice([-65504, 0, 3, 65504], (8, 256))]).astype(np.float16)
    codes, scale, low = D.quantise(x, levels, group)
    step = np.repeat(scale.astype(np.float64), group, -1)
    assert (np.abs(D.stands_for(codes, scale, low, group) - x.astype(np.float64)) <= step / 2).all()
    reach = x.astype(np.float64).reshape(len(x), -1, group)
    reach = reach.max(-1) - reach.min(-1)
    smaller = np.where(scale > 0, np.nextafter(scale, np.float16(-1)).astype(np.float64), 0)
    assert (scale.astype(np.float64) * levels >= reach).all() and ((smaller * levels < reach) | (scale == 0)).all()
