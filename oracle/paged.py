"""Serving a batch of sequences in numpy, float64: the position rotation in its layouts, the append to a paged
key-value cache, attention over it and the verification of drafted tokens. There is no counterpart in the
reference, whose cache is one contiguous sequence (`KVCache`, webtorch/_core.py:1543-1596) and whose greedy loop
picks on the host (`_pick`, webtorch/llm.py:1309-1336); the rotation in halves is `_rot`'s (webtorch/llm.py:1270-1304)."""
import numpy as np


def rotate(x, cos, sin, pairs=False, transpose=False):
    """x (.., H, HD) with angles cos, sin (.., rot / 2) -> the rotated rows, and per element the sum of the two products'
    magnitudes (for error bounds; 0 where a dimension is copied)."""
    x = np.asarray(x, np.float64)
    c, s = np.asarray(cos, np.float64)[..., None, :], np.asarray(sin, np.float64)[..., None, :]
    if transpose:
        s = -s
    R = c.shape[-1]
    ia, ib = (np.arange(0, 2 * R, 2), np.arange(1, 2 * R, 2)) if pairs else (np.arange(R), R + np.arange(R))
    a, b = x[..., ia], x[..., ib]
    y, mag = x.copy(), np.zeros_like(x)
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia], mag[..., ib] = np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)
    return y, mag


def rope(x, positions, cos, sin, pairs=False, transpose=False):
    """`rotate` by the tables' rows; a position outside them makes zeros."""
    p = np.asarray(positions)
    ok = (p >= 0) & (p < len(cos))
    at = np.where(ok, p, 0)
    y, mag = rotate(x, np.asarray(cos)[at], np.asarray(sin)[at], pairs, transpose)
    return np.where(ok[..., None, None], y, 0.0), mag


def slot_of(pos, table, page, num_pages):
    """(page, slot) of a position, None where there is none."""
    if pos < 0 or pos // page >= len(table) or not 0 <= table[pos // page] < num_pages:
        return None
    return int(table[pos // page]), int(pos % page)


def append(qkv, positions, pages, cache, n_heads, rope=None, qn=None, kn=None, eps=1e-6):
    """qkv (S, T, (NH + 2 NKV) HD), rope = (cos, sin, pairs) or None -> q (S, T, NH, HD), the new cache, both's magnitudes, and which
    slots (pages, page) were written."""
    num, _, nkv, page, hd = cache.shape
    S, T, _ = qkv.shape
    x = np.asarray(qkv, np.float64).reshape(S, T, n_heads + 2 * nkv, hd)
    out, qm = np.zeros((S, T, n_heads, hd)), np.zeros((S, T, n_heads, hd))
    full, cm, written = np.asarray(cache, np.float64).copy(), np.zeros(cache.shape), np.zeros((num, page), bool)
    for s in range(S):
        for t in range(T):
            pos = int(positions[s, t])
            at = slot_of(pos, pages[s], page, num)
            if at is None or (rope is not None and pos >= len(rope[0])):
                continue
            q, k, v = x[s, t, :n_heads], x[s, t, n_heads:n_heads + nkv], x[s, t, n_heads + nkv:]
            if qn is not None:
                q = q / np.sqrt((q * q).mean(-1, keepdims=True) + eps) * np.asarray(qn, np.float64)
            if kn is not None:
                k = k / np.sqrt((k * k).mean(-1, keepdims=True) + eps) * np.asarray(kn, np.float64)
            (q, a), (k, b) = (rotate(y, rope[0][pos], rope[1][pos], rope[2]) if rope is not None else (y, 0.0) for y in (q, k))
            out[s, t], qm[s, t] = q, np.maximum(a, np.abs(q))
            full[at[0], 0, :, at[1]], full[at[0], 1, :, at[1]], written[at] = k, v, True
            cm[at[0], 0, :, at[1]] = np.maximum(b, np.abs(k))
    return out, full, qm, cm, written


def attention(q, positions, pages, cache, scale=None):
    """q (S, T, NH, HD) -> the output, and per output an error scale: sum p |v|, and the largest sum |q k| scale of its row."""
    S, T, nh, hd = q.shape
    num, _, nkv, page, _ = cache.shape
    scale = hd ** -0.5 if scale is None else scale
    out, mag, top = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:3])
    for s in range(S):
        n = min(int(positions[s].max()) + 1, pages.shape[1] * page)
        at = [(p, slot_of(p, pages[s], page, num)) for p in range(max(n, 0))]
        at = [(p, a) for p, a in at if a is not None]
        if not at:
            continue
        where = np.array([p for p, _ in at])
        rows = cache[[a[0] for _, a in at], :, :, [a[1] for _, a in at]].astype(np.float64)  # (n, 2, NKV, HD)
        for t in range(T):
            m = int((where <= positions[s, t]).sum())
            if m == 0:
                continue
            for h in range(nh):
                k, v = rows[:m, 0, h * nkv // nh], rows[:m, 1, h * nkv // nh]
                x = q[s, t, h].astype(np.float64)
                a = k @ x * scale
                e = np.exp(a - a.max())
                p = e / e.sum()
                out[s, t, h], mag[s, t, h] = p @ v, p @ np.abs(v)
                top[s, t, h] = (np.abs(k) @ np.abs(x)).max() * abs(scale)
    return out, mag, top


def law(row, temperature):
    """The distribution of a row of logits, None where it has none."""
    x = np.asarray(row, np.float64)
    if not temperature > 0:
        x = np.where(np.isnan(x), -np.inf, x)
        if not (x > -np.inf).any():
            return None
        p = np.zeros(len(x))
        p[int(np.argmax(x))] = 1.0
        return p
    if np.isnan(x).any() or (x == np.inf).any() or not (x > -np.inf).any():
        return None
    e = np.exp((x - x.max()) / temperature)
    return e / e.sum()


def verify(logits, drafts, uniforms, draft_logits=None, temperature=1.0):
    """-> tokens (S, D + 1), accepted (S,), and per sequence how near (relative to the total) a border between tokens the draw fell."""
    S, rows, V = logits.shape
    D = rows - 1
    tokens, accepted, near = np.full((S, D + 1), -1, np.int32), np.zeros(S, np.int32), np.full(S, np.inf)
    for s in range(S):
        tau = float(np.broadcast_to(np.asarray(temperature, np.float64), (S,))[s])
        u = uniforms[s].astype(np.float64)
        i = 0
        while True:
            p = w = law(logits[s, i], tau)
            x = int(drafts[s, i]) if i < D else -1
            if x < 0:
                break
            q = np.zeros(V)
            if draft_logits is not None and tau > 0:
                q = law(draft_logits[s, i], tau)
            elif x < V:
                q[x] = 1.0
            if p is not None and x < V and q is not None and u[i] * q[x] < p[x]:
                tokens[s, i] = x
                i += 1
                continue
            if p is not None:
                w = np.maximum(p - q, 0.0) if q is not None and tau > 0 else p
            break
        accepted[s] = i
        if w is None:
            continue
        run = np.cumsum(w)
        if run[-1] == 0:
            tokens[s, i] = x if 0 <= x < V else -1
            continue
        want = u[D] * run[-1]
        hit = np.flatnonzero((run > want) & (w > 0))
        tokens[s, i] = hit[0] if len(hit) else np.flatnonzero(w > 0)[-1]
        near[s] = np.abs(run - want).min() / run[-1]
    return tokens, accepted, near
