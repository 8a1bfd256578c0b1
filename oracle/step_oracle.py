"""The calls of a speculative step restated plainly: whole numbers in Python loops, the rest in
float64 numpy.  Besides its result every attention or gradient function returns what a bound
on a float32 computation's error is made of (sums of magnitudes), so that the tests derive
their tolerances instead of guessing them.
"""
from __future__ import annotations

import numpy as np

U = 2.0 ** -24          # half a float32 step, relative


def parent_of(parent, i):
    return int(parent) if 0 <= int(parent) < i else -1


def ancestors(parents):
    """[n][n] bool: row i is set at i and at its ancestors."""
    n = len(parents)
    sees = np.zeros((n, n), bool)
    for i in range(n):
        j = i
        while j >= 0:
            sees[i, j] = True
            j = parent_of(parents[j], j)
    return sees


def pack_bits(sees, words):
    out = np.zeros((sees.shape[0], words), np.uint32)
    for i, j in zip(*np.nonzero(sees)):
        out[i, j // 32] |= np.uint32(1 << (j % 32))
    return out


def plan_step(lists, lengths, new, num_rows, max_new, block, index=None, parents=None, width=0, words=0, want_slots=False):
    B = len(lengths)
    starts, tables, totals = [0], np.zeros((B, max(width, 1)), np.int32), np.zeros(B, np.uint32)
    positions, slots = np.full(num_rows, -1, np.int32), np.full(num_rows, -1, np.int64)
    masks = np.zeros((num_rows, max(words, 1)), np.uint32)
    for b in range(B):
        n = min(max(int(new[b]), 0), max_new)
        start = min(starts[-1], num_rows)
        end = min(start + n, num_rows)
        n, length = end - start, max(int(lengths[b]), 0)
        starts.append(end)
        totals[b] = length + n
        row = int(index[b]) if index is not None else b
        entries = lists[row] if 0 <= row < len(lists) else []
        for j in range(min(width, len(entries), -(-(length + n) // block))):
            tables[b, j] = entries[j]
        if parents is not None:
            sees = ancestors(parents[start:end])
        else:
            sees = np.tri(n, n, dtype=bool)
        for i in range(n):
            depth = int(sees[i].sum()) - 1
            pos = length + depth
            positions[start + i] = pos
            page = pos // block
            if page < len(entries) and entries[page] >= 0:
                slots[start + i] = int(entries[page]) * block + pos % block
        if words:
            masks[start:end] = pack_bits(sees, words)
    return dict(starts=np.array(starts, np.int32), tables=tables, totals=totals, positions=positions, slots=slots, masks=masks)


def accept_tree(starts, parents, draft, target, lengths, num_rows, max_tree, max_path, tables=None, block=16):
    B = len(lengths)
    slots = np.full(num_rows, -1, np.int64)
    counts, nxt, totals = np.zeros(B, np.int32), np.full(B, -1, np.int32), np.zeros(B, np.uint32)
    path = np.full((B, max(max_path, 1)), -1, np.int32)
    for b in range(B):
        s = min(max(int(starts[b]), 0), num_rows)
        e = min(max(int(starts[b + 1]), s), num_rows)
        n, length = min(e - s, max_tree), max(int(lengths[b]), 0)
        depth, ok, best = [], [], -1
        for i in range(n):
            p = parent_of(parents[s + i], i)
            depth.append(0 if p < 0 else depth[p] + 1)
            ok.append(p < 0 or (ok[p] and int(draft[s + i]) == int(target[s + p])))
            if ok[i] and (best < 0 or depth[i] > depth[best]):
                best = i
        nodes = []
        j = best
        while j >= 0:
            nodes.append(j)
            j = parent_of(parents[s + j], j)
        nodes.reverse()
        counts[b], totals[b] = len(nodes), length + len(nodes)
        if nodes:
            nxt[b] = target[s + best]
        for d, j in enumerate(nodes):
            if d < max_path:
                path[b, d] = s + j
            if tables is not None:
                page, off = divmod(length + d, block)
                if page < tables.shape[1] and tables[b, page] >= 0:
                    slots[s + j] = int(tables[b, page]) * block + off
    return dict(slots=slots, counts=counts, path=path, next=nxt, totals=totals)


def _pair_index(dim, rotary, interleaved):
    """For every element: its angle, its partner and whether it is the first of its pair (rotary elements)."""
    half = rotary // 2
    d = np.arange(rotary)
    if interleaved:
        return d // 2, d ^ 1, d % 2 == 0
    return d % max(half, 1), np.where(d < half, d + half, d - half), d < half


def turned(x, positions, inv_freq, rotary, interleaved, sign=1.0):
    """x [rows][heads][dim] float64 with its first `rotary` elements turned by sign * angle."""
    if rotary == 0:
        return x.copy()
    angle = positions.astype(np.float64)[:, None] * inv_freq.astype(np.float64)
    which, other, first = _pair_index(x.shape[-1], rotary, interleaved)
    cos, sin = np.cos(angle)[:, which][:, None], sign * np.sin(angle)[:, which][:, None]
    y = x.copy()
    y[..., :rotary] = x[..., :rotary] * cos + np.where(first, -1.0, 1.0) * x[..., other] * sin
    return y


def pair_magnitude(x, rotary, interleaved):
    """|a| + |b| for rotated elements, |x| behind them."""
    m = np.abs(x)
    if rotary:
        _, other, _ = _pair_index(x.shape[-1], rotary, interleaved)
        m = m.copy()
        m[..., :rotary] = np.abs(x[..., :rotary]) + np.abs(x[..., other])
    return m


def norm_rotate(x, weight, positions, inv_freq, rotary, interleaved, eps):
    """(y, magnitude): the rotated norm and |a| + |b| of the values it is made of."""
    x, w = x.astype(np.float64), weight.astype(np.float64)
    n = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    return turned(n, positions, inv_freq, rotary, interleaved), pair_magnitude(n, rotary, interleaved)


def norm_rotate_backward(x, weight, dy, positions, inv_freq, rotary, interleaved, eps):
    """(dx, dw, magnitude of dx's terms, sum of |dn xhat|)."""
    x, w, dy = x.astype(np.float64), weight.astype(np.float64), dy.astype(np.float64)
    dn = turned(dy, positions, inv_freq, rotary, interleaved, -1.0)
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    xhat, g = x * r, dn * w
    dx = r * (g - xhat * (g * xhat).mean(-1, keepdims=True))
    size = pair_magnitude(dy, rotary, interleaved)
    magnitude = r * (np.abs(w) * size + np.abs(xhat) * (size * np.abs(w) * np.abs(xhat)).mean(-1, keepdims=True))
    return dx, (dn * xhat).sum((0, 1)), magnitude, (size * np.abs(xhat)).sum((0, 1))


def tree_attention(q, k, v, k_pool, v_pool, tables, lens, starts, block, masks=None, positions=None, window=0, max_new=1 << 30):
    """Rows [start_b, start_b+1) of q [rows][heads][dim] over the pages and their own rows.  Pools are
    [block][kv_head][slot][dim] float64 (dequantised).  Returns (out, weighted mean |v|, bound on a
    float32 score's error, number of keys); rows outside every request are NaN.  A key that a row
    does not see is left out of its sums altogether."""
    rows, H, D = q.shape
    KVH, G = k.shape[1], H // k.shape[1]
    out = np.full((rows, H, D), np.nan)
    mag, serr, count = np.zeros((rows, H, D)), np.zeros((rows, H)), np.zeros(rows, np.int64)
    pool_blocks = k_pool.shape[0]
    for b in range(len(lens)):
        s = min(max(int(starts[b]), 0), rows)
        e = min(max(int(starts[b + 1]), s), rows)
        n, length = min(e - s, max_new), int(lens[b])
        held = min(length, tables.shape[1] * block)
        tok = np.arange(held)
        blk = np.clip(tables[b][tok // block], 0, pool_blocks - 1) if held else np.zeros(0, int)
        ck, cv = k_pool[blk, :, tok % block], v_pool[blk, :, tok % block]          # [held][KVH][D]
        place = np.array([length + i if positions is None else max(int(positions[s + i]), length) for i in range(n)], np.int64)
        for i in range(n):
            if masks is None:
                sees = np.arange(n) <= i
            else:
                sees = np.array([(int(masks[s + i, j // 32]) >> (j % 32)) & 1 == 1 for j in range(n)], bool)
            cached = np.ones(held, bool)
            if window > 0:
                cached = tok > place[i] - window
                sees = sees & (place > place[i] - window)
            keys = np.concatenate([ck[cached], k[s:s + n][sees]]).astype(np.float64)
            vals = np.concatenate([cv[cached], v[s:s + n][sees]]).astype(np.float64)
            count[s + i] = len(keys)
            if len(keys) == 0:
                out[s + i] = 0.0
                continue
            for h in range(H):
                kk, vv, qq = keys[:, h // G], vals[:, h // G], q[s + i, h].astype(np.float64)
                with np.errstate(all="ignore"):
                    sc = kk @ qq / np.sqrt(D)
                    p = np.exp(sc - sc.max())
                    p /= p.sum()
                    out[s + i, h] = p @ vv
                    mag[s + i, h] = p @ np.abs(vv)
                    serr[s + i, h] = (D + 8) * U * (np.abs(kk) @ np.abs(qq)).max() / np.sqrt(D)
    return out, mag, serr, count
