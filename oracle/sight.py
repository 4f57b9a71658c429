"""Attention over a cache whose rows see a window or a tree, the tree's path, the cache moved together, and block tables: what
``include/et_abi.h`` says of et_mha_kv_window_f16, et_mha_kv_tree_f16, et_tree_*, et_kv_keep and et_kv_tables, in plain loops, numpy
and binary64."""
from __future__ import annotations

import numpy as np

from oracle.decode import GROUP, stands_for


def ways(parents, count):
    """Of each node, the nodes on its way up, itself included."""
    up = []
    for i in range(count):
        p = int(parents[i])
        up.append(([*up[p]] if 0 <= p < i else []) + [i])
    return up


def seen_words(parents, counts, n):
    """[B][n][words], zero in rows from counts[b] on."""
    out = np.zeros((len(parents), n, (n + 31) // 32), np.uint32)
    for b, row in enumerate(parents):
        for i, way in enumerate(ways(row, min(max(int(counts[b]), 0), n))):
            for j in way:
                out[b, i, j // 32] |= np.uint32(1 << (j % 32))
    return out


def window_sight(starts, counts, n, window, sinks, causal):
    """sees(b, i, positions) of et_mha_kv_window_f16."""
    def sees(b, i, pos):
        p = int(starts[b]) + i
        end = int(starts[b]) + min(max(int(counts[b]), 0), n)
        return (pos < (min(end, p + 1) if causal else end)) & ((pos > p - window) | (pos < sinks))
    return sees


def tree_sight(starts, counts, n, words, window, sinks):
    """sees(b, i, positions) of et_mha_kv_tree_f16."""
    def sees(b, i, pos):
        start, count = int(starts[b]), min(max(int(counts[b]), 0), n)
        bits = np.array([bool(words[b, i, j // 32] >> np.uint32(j % 32) & np.uint32(1)) for j in range(count)], bool)
        own = start + max(int(bits.sum()) - 1, 0)
        node = pos - start
        tree = (node >= 0) & (node < count) & bits[np.clip(node, 0, max(count - 1, 0))]
        near = (pos > own - window) | (pos < sinks) if window else np.ones(len(pos), bool)
        return ((node < 0) | tree) & near
    return sees


def attention(cache, table, starts, counts, Q, n, nh, scale, sees):
    """As oracle.decode.attention, of rows that see what `sees` says."""
    hd, per = cache.hd, nh // cache.nkv
    B = len(starts)
    Z, stepped, lows, reach = (np.full((B * n, nh * hd), np.nan) for _ in range(4))
    rep = lambda a: np.repeat(a.astype(np.float64), GROUP, -1)  # noqa: E731
    for b in range(B):
        count = min(max(int(counts[b]), 0), n)
        pos, k, v = cache.rows(table, b, int(starts[b]) + count)
        rows = slice(b * n, b * n + count)
        Z[rows] = stepped[rows] = lows[rows] = reach[rows] = 0
        if not len(pos):
            continue
        seen = np.array([sees(b, i, pos) for i in range(count)], bool).reshape(count, len(pos))
        key, size = stands_for(*k), rep(np.abs(k[1])) * k[0] + rep(np.abs(k[2]))
        step, low = rep(v[1]) * v[0], rep(v[2])
        for g in range(cache.nkv):
            ok = np.isfinite(key[:, g]).all(1) & np.isfinite(step[:, g] + low[:, g]).all(1)
            for h in range(g * per, (g + 1) * per):
                cols = slice(h * hd, (h + 1) * hd)
                q = Q[rows, cols].astype(np.float64)
                # rows that see only numbers, all at once; of others what they see is picked out
                whole = np.flatnonzero(seen.any(1) & ~(seen & ~ok).any(1) & np.isfinite(q).all(1))
                at, r = seen[np.ix_(whole, ok)], b * n + whole
                score = np.where(at, scale * (q[whole] @ key[ok, g].T), -np.inf)
                p = np.exp(score - score.max(1, keepdims=True, initial=-np.inf))
                p /= p.sum(1, keepdims=True)
                Z[r, cols] = p @ (step[ok, g] + low[ok, g])
                stepped[r, cols], lows[r, cols] = p @ step[ok, g], p @ np.abs(low[ok, g])
                reach[r, cols] = abs(scale) * np.where(at, np.abs(q[whole]) @ size[ok, g].T, 0).max(1, keepdims=True, initial=0)
                for i in np.setdiff1d(np.flatnonzero(seen.any(1)), whole):
                    at, r = seen[i], b * n + i
                    score = scale * (key[at, g] @ q[i])
                    p = np.exp(score - score.max())
                    p /= p.sum()
                    Z[r, cols] = p @ (step[at, g] + low[at, g])
                    stepped[r, cols], lows[r, cols] = p @ step[at, g], p @ np.abs(low[at, g])
                    reach[r, cols] = abs(scale) * (size[at, g] @ np.abs(q[i])).max()
    return Z, stepped, lows, reach


def follow(parents, tokens, choices, starts, counts, n):
    """path [B][n], kept, next tokens, next starts."""
    B = len(parents)
    path, kept, token = np.full((B, n), -1, np.int32), np.zeros(B, np.int32), np.full(B, -1, np.int32)
    for b in range(B):
        count = min(max(int(counts[b]), 0), n)
        now = 0 if count else None
        while now is not None:
            path[b, kept[b]] = now
            kept[b] += 1
            token[b] = choices[b][now]
            now = next((i for i in range(now + 1, count) if parents[b][i] == now and tokens[b][i] == token[b]), None)
    return path, kept, token, (np.asarray(starts, np.int64) + kept).astype(np.int32)


def keep(cache, table, starts, path, kept, n):
    """The host cache moved together: all places are read before any is written."""
    moves = []
    for b in range(len(starts)):
        for r in range(min(max(int(kept[b]), 0), n)):
            if not 0 <= path[b][r] < n:
                continue
            src, dst = cache.place(table, b, int(starts[b]) + int(path[b][r])), cache.place(table, b, int(starts[b]) + r)
            if src is None or dst is None:
                continue
            (p, o), at = src, dst
            moves.append((at, [cache.k_codes[p, :, o].copy(), cache.v_codes[p, :, o // 4, :, o % 4].copy(), cache.k_scales[p, :, :, o].copy(), cache.v_scales[p, :, :, o].copy()]))
    for (p, o), (kc, vc, ks, vs) in moves:
        cache.k_codes[p, :, o], cache.v_codes[p, :, o // 4, :, o % 4], cache.k_scales[p, :, :, o], cache.v_scales[p, :, :, o] = kc, vc, ks, vs


def tables(before, page, npages, starts, counts, shared, n, window, sinks, ring, state):
    """(table, ring, next state, slots) of et_kv_tables."""
    B, M = before.shape
    table, ring, head, free = before.copy(), ring.copy(), int(state[0]) % npages, min(max(int(state[1]), 0), npages)
    first = ring.copy()
    taken = given = missing = 0
    slots = np.full((B, n), -1, np.int64)
    for b in range(B):
        start, count = int(starts[b]), min(max(int(counts[b]), 0), n)
        for i in range(0 if shared is None else min(max(int(shared[b]), 0), M), M):
            needed = i * page < start + count and (not window or i * page < sinks or (i + 1) * page > start - window + 1)
            held = 0 <= before[b, i] < npages
            if held and not needed:
                if free + given < npages:
                    ring[(head + free + given) % npages] = before[b, i]
                given += 1
            if needed and not held:
                table[b, i] = first[(head + taken) % npages] if taken < free else -1
                missing += taken >= free
                taken += taken < free
            elif not needed:
                table[b, i] = -1
        for i in range(count):
            p = start + i
            if 0 <= p < M * page and 0 <= table[b, p // page] < npages:
                slots[b, i] = int(table[b, p // page]) * page + p % page
    return table, ring, np.array([(head + taken) % npages, min(free + given, npages) - taken, missing], np.int32), slots
