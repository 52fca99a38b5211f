"""Operators of a decoder's serving path, as cases that can be run and timed: per-head norms of queries
and keys with the position rotation and the cache write, attention over a key-value cache held in 4
bits, and log probabilities of given tokens with entropy and top alternatives.

`run` computes them in plain torch, or, where `own` is true, through this package's entry points.
`exact(case, seed)` gives the same outputs in float64, written apart.

The 4-bit cache is a uint8 tensor (NKV, blocks of 32 positions, 40 HD). A group of 32 consecutive
dimensions of one position's key (or value) row has two fp16 numbers S and Z, and a code c in 0 .. 15
stands for fp16(S (1 + c / 16) + Z). A block holds, one after the other: the key codes, 16 HD bytes; the
value codes, 16 HD bytes; (S, Z) of the keys, [position][group]; and of the values, [group][g][S of 8
positions, Z of 8 positions]. A 32-bit word has 8 codes, number e at bits 4 (e // 2) + 16 (e % 2):
8 dimensions 32 j + 8 g + e of the key of position 16 b + i, or dimension 16 t + i of the values of the
positions 16 (e // 4) + 4 g + e % 4. Words lie as [n // 4][g][i][n % 4] with n = b HD / 32 + j of
the keys, n = t of the values (i < 16, g < 4).
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
LIM = 16384.0  # magnitudes past it saturate in the 4-bit cache

# (query heads, key-value heads, head dimension): the 0.5B and 7B shapes of this repository's decoder
# configurations, a sparse-MoE decoder's with QK-norm, one key-value head per four query heads, no
# sharing, and wide heads
HEADS = ((14, 2, 64), (28, 4, 128), (32, 4, 128), (32, 8, 128), (8, 8, 64), (8, 2, 256))


# ---- the cases ------------------------------------------------------------------------
def listed():
    return [
        # one decoded token of a model with QK-norm: norms, rotation and the fp32 cache row; a call is latency
        dict(name="norm_rope_token", kind="norm_rope", cache="f32", NH=32, NKV=4, HD=128, T=1, pos=700, x="f32", norm=True),
        # a prompt of 700 tokens of the same model into the 4-bit cache, behind 133 cached positions (a block part full)
        dict(name="norm_rope_kv4_prompt700", kind="norm_rope", cache="kv4", NH=32, NKV=4, HD=128, T=700, pos=133, x="f32",
             norm=True),
        # a long prompt without QK-norm into the fp32 cache: the rotation alone
        dict(name="rope_prompt4001", kind="norm_rope", cache="f32", NH=28, NKV=4, HD=128, T=4001, pos=0, x="f32", norm=False),
        # one decoded token of the smallest decoder behind 700 positions
        dict(name="kv4_token_700", kind="attention", NH=14, NKV=2, HD=64, T=1, pos=700, x="f32"),
        # one decoded token at the end of a long context: the cache is read once
        dict(name="kv4_token_131000", kind="attention", NH=32, NKV=8, HD=128, T=1, pos=131000, x="f32"),
        # a chunk of 77 new tokens behind 30000 cached ones, fp16 rows
        dict(name="kv4_chunk77_30000", kind="attention", NH=32, NKV=8, HD=128, T=77, pos=30000, x="f16"),
        # a prompt of 2000 tokens of the 7B class from an empty cache, the engine's fp32 rows
        dict(name="kv4_prompt2000", kind="attention", NH=28, NKV=4, HD=128, T=2000, pos=0, x="f32"),
        # a long prompt, fp16 rows: the largest products
        dict(name="kv4_prompt6001_f16", kind="attention", NH=28, NKV=4, HD=128, T=6001, pos=0, x="f16"),
        # the probability of one decoded token with 5 alternatives, as a server reports it per token
        dict(name="logprobs_token", kind="logprobs", T=1, V=151936, pad=0, k=5, x="f32", masked=0.0),
        # a prompt of 700 tokens scored, 20 alternatives each
        dict(name="logprobs_prompt700", kind="logprobs", T=700, V=151936, pad=0, k=20, x="f32", masked=0.0),
        # 37 rows of fp16 logits in padded rows, a third of the vocabulary masked (constrained decoding)
        dict(name="logprobs_masked37", kind="logprobs", T=37, V=32003, pad=61, k=8, x="f16", masked=0.33),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm_rope", "attention", "attention", "logprobs"])
    x = rng.choice(["f32", "f32", "f16"])
    NH, NKV, HD = rng.choice(HEADS)
    if kind == "norm_rope":
        cache = rng.choice(["f32", "kv4", "kv4"])
        return dict(kind=kind, cache=cache, NH=NH, NKV=NKV, HD=HD, T=_log(rng, 1, 3900), pos=rng.choice([0, _log(rng, 1, 9000)]),
                    x=x if cache == "kv4" else "f32", norm=rng.random() < 0.7)
    if kind == "attention":
        T = rng.choice([1, 1, _log(rng, 2, 40), _log(rng, 2, 3000)])
        if T == 1:
            pos = _log(rng, 1, 120000)
        else:  # rows times keys stay below the largest listed case's
            pos = rng.choice([0, _log(rng, 1, min(60000, 200000000 // (NH * T)))])
        return dict(kind=kind, NH=NH, NKV=NKV, HD=HD, T=T, pos=pos, x=x)
    V = rng.choice([151936, 152064, 128256, rng.randint(1000, 150000)])
    return dict(kind=kind, T=_log(rng, 1, max(2, 95000000 // V)), V=V, pad=rng.choice([0, rng.randint(1, 64)]), k=rng.randint(0, 20), x=x,
                masked=rng.choice([0.0, 0.0, rng.uniform(0.05, 0.95)]))


# ---- inputs ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000003 + 29)
    return g


def _dtype(s):
    return torch.float16 if s == "f16" else torch.float32


def _heads(g, n, HD, rows):
    """(rows, n, HD) values N(0, 1) with one channel in 32 of each head four times as large, as keys have."""
    big = 1.0 + 3.0 * (torch.rand((n, HD), device=DEV, generator=g) < 1 / 32).float()
    return torch.randn((rows, n, HD), device=DEV, generator=g) * big


def _tables(HD, n):
    inv = 1.0 / (1e6 ** (np.arange(0, HD, 2, dtype=np.float64) / HD))
    ang = torch.from_numpy(np.arange(n, dtype=np.float64)).to(DEV)[:, None] * torch.from_numpy(inv).to(DEV)[None, :]
    return torch.cos(ang).float(), torch.sin(ang).float()


def _codes(x):
    """Codes, S and Z of rows x (..., HD) fp32 as the 4-bit cache holds them."""
    xg = x.unflatten(-1, (-1, 32))
    fine = torch.isfinite(xg).all(-1, keepdim=True)
    xc = xg.clamp(-LIM, LIM)
    lo, hi = xc.amin(-1, keepdim=True), xc.amax(-1, keepdim=True)
    # a tensor divisor: torch multiplies by the reciprocal of a number
    S = torch.maximum((hi - lo) * 16.0 / torch.full_like(lo, 15.0), lo.abs() / 128.0).half()
    Z = (lo - S.float()).half()
    t = torch.where(S > 0, (xc - Z.float()) / S.float() * 16.0, torch.full_like(xc, 16.0))
    c = (t.round() - 16.0).clamp(0.0, 15.0)
    nan = torch.full_like(S, float("nan"))
    S, Z = torch.where(fine, S, nan), torch.where(fine, Z, nan)
    return torch.where(fine, c, torch.zeros_like(c)).to(torch.uint8), S, Z


def _stands_for(c, S, Z):
    return (S.float() * (1.0 + c.float() / 16.0) + Z.float()).half().float().flatten(-2)


def _words(c):
    """(..., 8) codes as one 32-bit word each."""
    sh = torch.tensor([4 * (e // 2) + 16 * (e % 2) for e in range(8)], device=c.device)
    w = (c.long() << sh).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _pack(k, v):
    """Rows (positions, NKV, HD) fp32 of keys and values as a 4-bit cache of whole blocks."""
    n, NKV, HD = k.shape
    NB, NT = (n + 31) // 32, HD // 16
    parts = []
    for x, value in ((k, False), (v, True)):
        x = torch.cat([x, x.new_zeros((32 * NB - n, NKV, HD))]).transpose(0, 1)
        c, S, Z = _codes(x)
        if value:
            w = _words(c.reshape(NKV, NB, 2, 4, 4, NT, 16).permute(0, 1, 5, 3, 6, 2, 4).flatten(-2))
            m = torch.stack([S, Z], 0).reshape(2, NKV, NB, 2, 4, 4, HD // 32).permute(1, 2, 6, 4, 0, 3, 5)
        else:
            w = _words(c.reshape(NKV, NB, 2, 16, HD // 32, 4, 8)).permute(0, 1, 2, 4, 5, 3)
            m = torch.stack([S, Z], -1)
        w = w.reshape(NKV, NB, NT // 4, 4, 64).transpose(3, 4).contiguous()
        parts.append((w.view(torch.uint8).reshape(NKV, NB, 16 * HD), m.contiguous().view(torch.uint8).reshape(NKV, NB, 4 * HD)))
    (kw, km), (vw, vm) = parts
    return torch.cat([kw, vw, km, vm], 2).contiguous()


def _unpack(cache, n):
    """fp32 keys and values (NKV, n, HD) that a 4-bit cache stands for."""
    NKV, NB, HD = cache.shape[0], cache.shape[1], cache.shape[2] // 40
    NT = HD // 16
    sh = torch.tensor([4 * (e // 2) + 16 * (e % 2) for e in range(8)], device=cache.device, dtype=torch.int32)
    at = lambda a, b, t: cache[:, :, a * HD:b * HD].contiguous().view(t)  # noqa: E731
    codes = lambda w: (w.reshape(NKV, NB, NT // 4, 64, 4).transpose(3, 4).reshape(-1, 1) >> sh) & 15  # noqa: E731
    kc = codes(at(0, 16, torch.int32)).reshape(NKV, NB, 2, HD // 32, 4, 16, 8).permute(0, 1, 2, 5, 3, 4, 6).reshape(NKV, 32 * NB, -1, 32)
    vc = codes(at(16, 32, torch.int32)).reshape(NKV, NB, NT, 4, 16, 2, 4).permute(0, 1, 5, 3, 6, 2, 4).reshape(NKV, 32 * NB, -1, 32)
    km = at(32, 36, torch.float16).reshape(NKV, 32 * NB, HD // 32, 2, 1)
    vm = at(36, 40, torch.float16).reshape(NKV, NB, HD // 32, 4, 2, 2, 4).permute(4, 0, 1, 5, 3, 6, 2).reshape(2, NKV, 32 * NB, HD // 32, 1)
    return _stands_for(kc, km[..., 0, :], km[..., 1, :])[:, :n], _stands_for(vc, vm[0], vm[1])[:, :n]


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["kind"] == "logprobs":
        T, V, pad = c["T"], c["V"], c["pad"]
        # rows from flat to peaked, as positions of a text are
        x = torch.randn((T, V + pad), device=DEV, generator=g) * (1.0 + 2.0 * torch.rand((T, 1), device=DEV, generator=g))
        ids = torch.randint(0, V, (T,), device=DEV, generator=g, dtype=torch.int32)
        likely = torch.rand(T, device=DEV, generator=g) < 0.7  # most given tokens are likely ones
        x[torch.arange(T, device=DEV), ids.long()] += torch.where(likely, 8.0, 0.0)
        if c["masked"]:
            x[:, torch.rand(V + pad, device=DEV, generator=g) < c["masked"]] = -math.inf
        return {"case": c, "logits": x.to(_dtype(c["x"]))[:, :V], "ids": ids}
    NH, NKV, HD, T, pos = c["NH"], c["NKV"], c["HD"], c["T"], c["pos"]
    state = torch.tensor([pos, 0, 0, 0], dtype=torch.int32, device=DEV)
    n = pos + T
    if c["kind"] == "attention":
        q = torch.randn((T, NH, HD), device=DEV, generator=g)
        k, v = _heads(g, NKV, HD, n), torch.randn((n, NKV, HD), device=DEV, generator=g)
        return {"case": c, "q": q.to(_dtype(c["x"])), "cache": _pack(k, v), "state": state}
    qkv = torch.cat([_heads(g, NH, HD, T), _heads(g, NKV, HD, T), torch.randn((T, NKV, HD), device=DEV, generator=g)], 1)
    cos, sin = _tables(HD, n if c["cache"] == "f32" else (n + 31) // 32 * 32)  # a row per position of the cache
    st = {"case": c, "qkv": qkv.reshape(T, -1).to(_dtype(c["x"])), "state": state, "cos": cos, "sin": sin, "qn": None, "kn": None}
    if c["norm"]:
        st["qn"], st["kn"] = (1.0 + 0.2 * torch.randn(HD, device=DEV, generator=g) for _ in range(2))
    if c["cache"] == "f32":
        st["kc"], st["vc"] = (torch.zeros((NKV, n, HD), device=DEV) for _ in range(2))
    else:
        st["cache"] = torch.zeros((NKV, (n + 31) // 32, 40 * HD), dtype=torch.uint8, device=DEV)
    return st


# ---- one pass -------------------------------------------------------------------------
def _norm_rope(x, w, cos, sin):
    """x (T, heads, HD) of any float type, in that type."""
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.to(x.dtype)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _run_norm_rope(s):
    c = s["case"]
    NH, NKV, HD, T, pos = c["NH"], c["NKV"], c["HD"], c["T"], c["pos"]
    if own:
        from webpytorch_amd import core
        if c["cache"] == "f32":
            q = core.qk_norm_rope(s["qkv"], s["state"], s["cos"], s["sin"], NH, (s["kc"], s["vc"]), qn=s["qn"], kn=s["kn"])
            return {"q": q, "k": s["kc"], "v": s["vc"]}
        q = core.qk_norm_rope(s["qkv"], s["state"], s["cos"], s["sin"], NH, s["cache"], qn=s["qn"], kn=s["kn"])
        k, v = core.kv4_dequant(s["cache"], pos, T)
        return {"q": q, "k": k, "v": v}
    wide = torch.float32 if c["cache"] == "f32" else torch.float64  # codes go by which side of a border a key is on
    x = s["qkv"].reshape(T, NH + 2 * NKV, HD)
    cos, sin = (t[pos:pos + T, None].to(wide) for t in (s["cos"], s["sin"]))
    q = _norm_rope(x[:, :NH].to(wide), s["qn"], cos, sin).to(x.dtype)
    k = _norm_rope(x[:, NH:NH + NKV].to(wide), s["kn"], cos, sin).float().transpose(0, 1)
    v = x[:, NH + NKV:].float().transpose(0, 1)
    if c["cache"] == "f32":
        s["kc"][:, pos:pos + T], s["vc"][:, pos:pos + T] = k, v
        return {"q": q, "k": s["kc"], "v": s["vc"]}
    return {"q": q, "k": _stands_for(*_codes(k)), "v": _stands_for(*_codes(v))}


def _run_attention(s):
    c = s["case"]
    NH, NKV, HD, T, pos = c["NH"], c["NKV"], c["HD"], c["T"], c["pos"]
    if own:
        from webpytorch_amd import core
        return core.attention_kv4(s["q"], s["cache"], s["state"])
    rep, n = NH // NKV, pos + T
    k, v = _unpack(s["cache"], n)
    q = s["q"].float().reshape(T, NKV, rep, HD).permute(1, 2, 0, 3).reshape(NKV, rep * T, HD)
    a = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(1.0 / math.sqrt(HD)).reshape(NKV, rep, T, n)
    if T > 1:
        later = torch.arange(n, device=DEV)[None, :] > pos + torch.arange(T, device=DEV)[:, None]
        a.masked_fill_(later, -math.inf)
    a = (a - a.amax(-1, keepdim=True)).exp_()
    a = a / a.sum(-1, keepdim=True)
    o = torch.matmul(a.reshape(NKV, rep * T, n), v)
    return o.reshape(NKV, rep, T, HD).permute(2, 0, 1, 3).reshape(T, NH, HD).to(s["q"].dtype)


def _order(x):
    """64-bit keys in the order of alternatives: the larger value first, of equal ones the lower index; NaN last."""
    x = torch.where(torch.isnan(x), -math.inf, x) + 0.0
    b = x.view(torch.int32)
    b = torch.where(b < 0, b ^ 0x7FFFFFFF, b).long()
    return (b << 32) | (0xFFFFFFFF - torch.arange(x.shape[1], device=x.device))


def _run_logprobs(s):
    c = s["case"]
    if own:
        from webpytorch_amd import core
        r = core.token_logprobs(s["logits"], s["ids"], c["k"])
        return {"logprobs": r.logprobs, "entropy": r.entropy, "ranks": r.ranks, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs}
    x = s["logits"].float()
    xt = x.gather(1, s["ids"].long()[:, None])
    m = x.amax(1, keepdim=True)
    d = x - m
    e = d.exp()
    z = e.sum(1)
    lse = m[:, 0] + z.log()
    entropy = z.log() - torch.where(e > 0, e * d, 0.0).sum(1) / z
    top = 0xFFFFFFFF - (_order(x).topk(c["k"], 1).values & 0xFFFFFFFF)
    return {"logprobs": xt[:, 0] - lse, "entropy": entropy, "ranks": (x > xt).sum(1).to(torch.int32), "top_ids": top.to(torch.int32),
            "top_logprobs": x.gather(1, top) - lse[:, None]}


def run(state):
    return {"norm_rope": _run_norm_rope, "attention": _run_attention, "logprobs": _run_logprobs}[state["case"]["kind"]](state)


def work(case):
    c = case
    size = 2 if c["x"] == "f16" else 4
    if c["kind"] == "logprobs":
        n = c["T"] * c["V"]
        return {"bytes": n * size + c["T"] * (16 + 8 * c["k"]), "flops": 5 * n}
    NH, NKV, HD, T, pos = c["NH"], c["NKV"], c["HD"], c["T"], c["pos"]
    if c["kind"] == "attention":  # 5 bits a value, a key and a value row per position and head
        return {"bytes": (pos + T) * NKV * HD * 1.25 + 2 * T * NH * HD * size,
                "flops": 4 * NH * HD * sum(pos + t + 1 for t in range(T))}
    # the cache rows, and for the 4-bit one the values they stand for, which the pass returns
    rows = 2 * NKV * HD * 4 if c["cache"] == "f32" else 2 * NKV * HD * (0.625 + 4)
    return {"bytes": T * (((NH + 2 * NKV) + NH) * HD * size + rows + HD * 4), "flops": T * (NH + NKV) * HD * 9}


# ---- the same in float64 ----------------------------------------------------------------
def _exact_group(x):
    """What the 4-bit cache stands for, rows x (..., HD) float64 holding fp32 values, by its rule."""
    f = x.float().reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    f = torch.minimum(torch.maximum(f, f.new_tensor(-LIM)), f.new_tensor(LIM))
    lo = f.min(-1, keepdim=True).values
    step16 = torch.maximum((f.max(-1, keepdim=True).values - lo) * 16 / torch.full_like(lo, 15), lo.abs() * 2.0 ** -7).to(torch.float16)
    zero = (lo - step16.float()).to(torch.float16)
    ratio = torch.nan_to_num((f - zero.float()) / step16.float(), nan=1.0, posinf=1.0, neginf=1.0)
    code = torch.clamp(torch.round(ratio * 16) - 16, 0, 15).double()
    return (step16.double() * (16 + code) / 16 + zero.double()).float().half().double().reshape(x.shape)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "logprobs":
        x = s["logits"].double()
        lse = torch.logsumexp(x, 1)
        lp = x - lse[:, None]
        p = lp.exp()
        entropy = -(p * torch.nan_to_num(lp, neginf=0.0)).sum(1)
        at = s["ids"].long()[:, None]
        top = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["k"]]
        return {"logprobs": lp.gather(1, at)[:, 0], "entropy": entropy, "ranks": (x > x.gather(1, at)).sum(1).int(), "top_ids": top.int(),
                "top_logprobs": lp.gather(1, top)}
    NH, NKV, HD, T, pos = c["NH"], c["NKV"], c["HD"], c["T"], c["pos"]
    rep = NH // NKV
    if c["kind"] == "attention":
        k, v = (t.double() for t in _unpack(s["cache"], pos + T))
        q = s["q"].double()
        out = torch.empty_like(q)
        upto = pos + torch.arange(T, device=DEV)
        for h in range(NH):
            a = torch.mm(q[:, h], k[h // rep].t().contiguous()) / math.sqrt(HD)
            a[torch.arange(pos + T, device=DEV)[None, :] > upto[:, None]] = -math.inf
            out[:, h] = torch.mm(torch.softmax(a, 1), v[h // rep])
        return out
    x = s["qkv"].double().reshape(T, NH + 2 * NKV, HD)
    turn = torch.complex(s["cos"][pos:pos + T].double(), s["sin"][pos:pos + T].double())[:, None]
    rows = []
    for part, w in ((x[:, :NH], s["qn"]), (x[:, NH:NH + NKV], s["kn"])):
        if w is not None:
            part = part * torch.rsqrt(part.pow(2).sum(-1, keepdim=True) / HD + 1e-6) * w.double()
        z = torch.complex(part[..., :HD // 2].contiguous(), part[..., HD // 2:].contiguous()) * turn
        rows.append(torch.cat([z.real, z.imag], -1))
    k, v = rows[1].transpose(0, 1), x[:, NH + NKV:].transpose(0, 1)
    if c["cache"] == "kv4":
        return {"q": rows[0], "k": _exact_group(k), "v": _exact_group(v)}
    full = [torch.zeros((NKV, pos + T, HD), dtype=torch.float64, device=DEV) for _ in range(2)]
    full[0][:, pos:], full[1][:, pos:] = k, v
    return {"q": rows[0], "k": full[0], "v": full[1]}
