"""Decoding from a cache of keys and values in 4 or 8 bits, and 4-bit weights: the formats of ``include/et_abi.h`` (et_kv_cache,
et_linear_w4_f16) and what is computed from them, in numpy and binary64."""
from __future__ import annotations

import numpy as np

GROUP = 32
F16 = np.arange(0x7C00, dtype=np.uint16).view(np.float16).astype(np.float64)  # the finite binary16 numbers from zero up


def quantise(x, levels, group=GROUP):
    """binary16 [..., channels] -> codes uint8 [..., channels], scale and low binary16 [..., channels / group]."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, group)
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], 0.0, g)
    low, reach = g.min(-1), g.max(-1) - g.min(-1)
    scale = F16[np.searchsorted(F16 * levels, reach)]  # the first whose steps reach that far
    codes = np.rint((g - low[..., None]) / np.where(scale > 0, scale, 1.0)[..., None])
    assert codes.max(initial=0) <= levels
    return (codes.astype(np.uint8).reshape(x.shape), scale.astype(np.float16), np.where(bad, np.nan, low).astype(np.float16))


def stands_for(codes, scale, low, group=GROUP):
    """low + scale * code in binary64."""
    rep = lambda a: np.repeat(a.astype(np.float64), group, -1)  # noqa: E731
    return rep(low) + rep(scale) * codes.astype(np.float64)


def to_f16(x):
    return np.minimum(x, 65504.0).astype(np.float32).astype(np.float16)


class Cache:
    """The buffers of a cache on the host; rows are written in a plain loop."""

    def __init__(self, bits, nkv, hd, page, npages, fill=0xA5):
        self.bits, self.nkv, self.hd, self.page, self.npages, self.levels = bits, nkv, hd, page, npages, 2 ** bits - 1
        self.k_codes = np.full((npages, nkv, page, hd * bits // 8), fill, np.uint8)
        self.v_codes = np.full((npages, nkv, page // 4, hd * bits // 16, 4), fill * 0x101, np.uint16)
        self.k_scales = np.full((npages, nkv, hd // GROUP, page, 2), np.nan, np.float16)
        self.v_scales = self.k_scales.copy()

    def place(self, table, b, pos):
        """Page and offset of a position, or None."""
        if pos < 0 or pos // self.page >= table.shape[1]:
            return None
        p = int(table[b, pos // self.page])
        return (p, pos % self.page) if 0 <= p < self.npages else None

    def _bytes(self, codes):
        return codes if self.bits == 8 else codes[..., 0::2] | codes[..., 1::2] << 4

    def _codes(self, data):
        return data if self.bits == 8 else np.stack([data & 15, data >> 4], -1).reshape(*data.shape[:-1], -1)

    def write(self, table, starts, counts, K, V, n):
        kq, vq = (quantise(x.reshape(-1, self.nkv, self.hd), self.levels) for x in (K, V))
        for b in range(len(starts)):
            for i in range(min(max(int(counts[b]), 0), n)):
                at = self.place(table, b, int(starts[b]) + i)
                if at is None:
                    continue
                p, o = at
                r = b * n + i
                self.k_codes[p, :, o] = self._bytes(kq[0][r])
                self.v_codes[p, :, o // 4, :, o % 4] = np.ascontiguousarray(self._bytes(vq[0][r])).view(np.uint16)
                for scales, q in ((self.k_scales, kq), (self.v_scales, vq)):
                    scales[p, :, :, o, 0], scales[p, :, :, o, 1] = q[1][r], q[2][r]

    def token(self, p, o):
        """(codes, scale, low) of keys and of values, each [nkv][...], of one place."""
        v = np.ascontiguousarray(self.v_codes[p, :, o // 4, :, o % 4]).view(np.uint8)
        return [(self._codes(data), s[p, :, :, o, 0], s[p, :, :, o, 1]) for data, s in ((self.k_codes[p, :, o], self.k_scales), (v, self.v_scales))]

    def rows(self, table, b, end):
        """Positions of sequence b that have a place below end, and their (codes, scale, low) of keys and of values, stacked."""
        places = [(pos, self.place(table, b, pos)) for pos in range(max(0, end))]
        places = [(pos, at) for pos, at in places if at is not None]
        got = [self.token(*at) for _, at in places]
        stack = lambda kv: tuple(np.stack([g[kv][j] for g in got]) for j in range(3)) if got else None  # noqa: E731
        return np.array([pos for pos, _ in places], np.int64), stack(0), stack(1)


def attention(cache, table, starts, counts, Q, n, nh, scale, causal):
    """Z [B * n][nh * hd] in binary64 (NaN in rows from counts[b] on), and for every value the parts that roundings act on: the sum
    of p |scale * code| and of p |low| over the sum of p, and how far the row's scores may be from exact ones for every 2^-24 of
    rounding: the largest over the keys of sum |q| |key| * scale."""
    hd, per = cache.hd, nh // cache.nkv
    B = len(starts)
    Z, stepped, lows, reach = (np.full((B * n, nh * hd), np.nan) for _ in range(4))
    for b in range(B):
        count = min(max(int(counts[b]), 0), n)
        end = int(starts[b]) + count
        pos, k, v = cache.rows(table, b, end)
        for i in range(count):
            r = b * n + i
            upto = int(starts[b]) + i + 1 if causal else end
            seen = pos < upto
            if not seen.any():
                Z[r] = stepped[r] = lows[r] = reach[r] = 0
                continue
            for h in range(nh):
                g, cols = h // per, slice(h * hd, (h + 1) * hd)
                q = Q[r, cols].astype(np.float64)
                key = stands_for(*(a[seen, g] for a in k))
                vc, vs, vl = (a[seen, g].astype(np.float64) for a in v)
                score = scale * (key @ q)
                p = np.exp(score - score.max())
                p /= p.sum()
                step, low = np.repeat(vs, GROUP, -1) * vc, np.repeat(vl, GROUP, -1)
                Z[r, cols] = p @ (step + low)
                stepped[r, cols], lows[r, cols] = p @ step, p @ np.abs(low)
                ks, kl = (np.repeat(np.abs(a[seen, g].astype(np.float64)), GROUP, -1) for a in k[1:])
                reach[r, cols] = abs(scale) * ((ks * k[0][seen, g] + kl) @ np.abs(q)).max()
    return Z, stepped, lows, reach


def w4_pack(W, group):
    codes, scale, low = quantise(W, 15, group)
    return codes[:, 0::2] | codes[:, 1::2] << 4, np.ascontiguousarray(np.stack([scale, low], -1).transpose(1, 0, 2))


def w4_dense(codes, scales, group):
    """The weight in binary64."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)
    return stands_for(c, scales[..., 0].T, scales[..., 1].T, group)
