"""The 4-bit key-value cache, attention over it, QK-norm with RoPE and token log probabilities, restated in
numpy (test infrastructure only; see `oracle/__init__.py`). The cache's codes are defined by fp32 operations,
done here in numpy float32; everything else is float64.

Pins: the layout and the rule are those of `include/miq.h`; the rule's own error bound and the layout's
round trip are checked by `tests/test_oracle_kv4.py`."""
import numpy as np

GROUP, BLOCK, LIMIT = 32, 32, np.float32(16384)


def quantize(x):
    """codes (..., HD) and S, Z (..., HD / 32) float16 of rows x (..., HD) float32."""
    g = np.asarray(x, np.float32).reshape(x.shape[:-1] + (-1, GROUP))
    bad = ~np.isfinite(g).all(-1)
    g = np.clip(np.where(bad[..., None], np.float32(0), g), -LIMIT, LIMIT)
    lo, hi = g.min(-1), g.max(-1)
    S = np.maximum((hi - lo) * np.float32(16) / np.float32(15), np.abs(lo) / np.float32(128)).astype(np.float16)
    Z = (lo - S.astype(np.float32)).astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        r = (g - Z.astype(np.float32)[..., None]) / S.astype(np.float32)[..., None]
    c = np.clip(np.rint(r * np.float32(16)) - np.float32(16), 0, 15)
    c = np.where((S > 0)[..., None], c, 0).astype(np.uint8)
    return c.reshape(x.shape), np.where(bad, np.float16("nan"), S), np.where(bad, np.float16("nan"), Z)


def stands_for(c, S, Z):
    """float64 values (each an fp16 number) of codes c (..., HD)."""
    g = c.reshape(c.shape[:-1] + (-1, GROUP)).astype(np.float64)
    v = S.astype(np.float64)[..., None] * (1 + g / 16) + Z.astype(np.float64)[..., None]
    return v.astype(np.float16).astype(np.float64).reshape(c.shape)


def _places(HD):
    """Byte of the word and bit of the code in a record, [position][dimension], of keys and of values, and
    the bytes of S and Z, [position][group]."""
    p, d = np.meshgrid(np.arange(BLOCK), np.arange(HD), indexing="ij")
    word = lambda n, g, i: (((n // 4) * 64 + g * 16 + i) * 4 + n % 4) * 4  # noqa: E731
    bit = lambda e: 4 * (e // 2) + 16 * (e % 2)  # noqa: E731
    key = word((p // 16) * (HD // 32) + d // 32, d % 32 // 8, p % 16), bit(d % 8)
    g, e = p % 16 // 4, 4 * (p // 16) + p % 4
    value = 16 * HD + word(d // 16, g, d % 16), bit(e)
    pg, j = np.meshgrid(np.arange(BLOCK), np.arange(HD // 32), indexing="ij")
    km = 32 * HD + (pg * (HD // 32) + j) * 4
    vm = 36 * HD + ((j * 4 + pg % 16 // 4) * 16 + 4 * (pg // 16) + pg % 4) * 2
    return key, value, (km, km + 2), (vm, vm + 16)


def unpack(cache, n):
    """(codes, S, Z) of the keys and of the values of positions 0 .. n - 1, cache (NKV, blocks, 40 HD) uint8."""
    NKV, NB, rec = cache.shape
    HD = rec // 40
    out = []
    for (w, b), (ms, mz) in zip(_places(HD)[:2], _places(HD)[2:]):
        at = lambda i, k: cache[:, :, i + k].astype(np.uint32) << np.uint32(8 * k)  # noqa: E731
        words = at(w, 0) | at(w, 1) | at(w, 2) | at(w, 3)
        c = ((words >> b.astype(np.uint32)) & 15).astype(np.uint8).reshape(NKV, NB * BLOCK, HD)
        half = lambda i: (at(i, 0) | at(i, 1)).astype(np.uint16).view(np.float16).reshape(NKV, NB * BLOCK, -1)  # noqa: E731
        out.append(tuple(t[:, :n] for t in (c, half(ms), half(mz))))
    return out


def norm_rope(x, w, cos, sin, eps=1e-6):
    """float64 (T, heads, HD) of rows x, cos / sin (T, HD / 2)."""
    x = np.asarray(x, np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    h = x.shape[-1] // 2
    c, s = (np.asarray(t, np.float64)[:, None] for t in (cos, sin))
    return np.concatenate([x[..., :h] * c - x[..., h:] * s, x[..., h:] * c + x[..., :h] * s], -1)


def attention(q, k, v, pos, scale):
    """float64 causal GQA: q (T, NH, HD), k and v (NKV, n, HD); rows without a key are zero."""
    T, NH, HD = q.shape
    rep, n = NH // k.shape[0], k.shape[1]
    out = np.zeros((T, NH, HD))
    for t in range(T):
        S = min(pos + t + 1, n)
        if S <= 0:
            continue
        for h in range(NH):
            s = k[h // rep, :S].astype(np.float64) @ q[t, h].astype(np.float64) * scale
            p = np.exp(s - s.max())
            out[t, h] = (p / p.sum()) @ v[h // rep, :S].astype(np.float64)
    return out


def token_logprobs(x, ids, k):
    """(logprobs, entropy, ranks, top_ids, top_logprobs) in float64 of rows x (T, V)."""
    x = np.asarray(x).astype(np.float64)
    T, V = x.shape
    out = [np.zeros(T), np.zeros(T), np.full(T, -1), np.zeros((T, k), np.int64), np.zeros((T, k))]
    for t in range(T):
        r, m = x[t], np.nanmax(np.append(x[t], -np.inf))
        with np.errstate(invalid="ignore", divide="ignore"):
            lp = np.full(V, -np.inf) if m == -np.inf and not np.isnan(r).any() else r - m - np.log(np.exp(r - m).sum())
            if np.isnan(r).any() or m == np.inf:
                lp = np.full(V, np.nan)
            p = np.exp(lp)
            out[1][t] = -np.where(p == 0, 0, p * np.where(p == 0, 0, lp)).sum()
        if 0 <= ids[t] < V:
            out[0][t], out[2][t] = lp[ids[t]], (r > r[ids[t]]).sum()
        o = np.argsort(-np.where(np.isnan(r), -np.inf, r), kind="stable")[:k]
        out[3][t], out[4][t] = o, lp[o]
    return out
