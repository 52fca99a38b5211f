"""Operators of serving a batch of sequences from a paged key-value cache, as cases that can be run and
timed: the position rotation in its layouts, the rotation with the append to the cache, attention of the new
tokens over it, and the verification of drafted tokens.

`run` computes them in plain torch, or, where `own` is true, through this package's entry points.
`exact(case, seed)` gives the same outputs in float64, written apart.

A cache is one tensor (pages, 2, NKV, P, HD): keys at [:, 0], values at [:, 1]. Position n of sequence s lies in slot
n % P of page pages[s, n // P] (int32, -1: none). A batch has S sequences of T new tokens at positions[s, t] (int32,
-1: no token).

Drafted tokens: token i of a sequence has the target's logits row i and the draft's; p and q are their
softmaxes at the temperature. Token x_i is accepted while u_i q_i(x_i) < p_i(x_i); at the first that is not, a token is
drawn from max(p_i - q_i, 0), behind the last one from p: the first index whose running sum passes u_D times the
total. A draft that is no distribution of its own (no draft logits) has q_i(x_i) = 1. At temperature 0 p is all at the largest logit.
"""
import math

import torch

own = False

DEV = "cuda"

# (query heads, key-value heads, head dimension): the 0.5B and 7B shapes of this repository's decoder
# configurations, a sparse-MoE decoder's with QK-norm, one key-value head per four query heads, no
# sharing, and wide heads
HEADS = ((14, 2, 64), (28, 4, 128), (32, 4, 128), (32, 8, 128), (8, 8, 64), (8, 2, 256))
PAGES = (16, 32, 64, 128, 256)


# ---- the cases ------------------------------------------------------------------------
def listed():
    return [
        # queries of one decoded token of 64 sequences at far positions: a call is latency
        dict(name="rope_batch64", kind="rope", T=64, H=32, HD=128, rot=128, layout="half", scale="yarn", ctx=131072, x="f32", transpose=False,
             pad=0),
        # the query heads within the fused q|k|v rows of a long prompt, the first half of each head rotated in neighbouring pairs
        dict(name="rope_prompt7001_partial", kind="rope", T=7001, H=32, HD=128, rot=64, layout="pairs", scale="none", ctx=8192, x="f16",
             transpose=False, pad=2048),
        # the gradient of a rotation stretched to a longer context
        dict(name="rope_gradient4001", kind="rope", T=4001, H=28, HD=128, rot=128, layout="half", scale="linear", ctx=32768, x="f32",
             transpose=True, pad=0),
        # the new token of each of 64 sequences of up to 700 positions: norms, rotation, append
        dict(name="append_batch64", kind="append", S=64, T=1, NH=32, NKV=4, HD=128, P=64, most=700, rot=128, layout="half", norm=True,
             x="f32", cache="f16"),
        # four prompts of 300 to 1500 tokens in one padded batch, rotated in neighbouring pairs, into an fp32 cache
        dict(name="append_prompts4x1500", kind="append", S=4, T=1500, NH=28, NKV=4, HD=128, P=16, most=0, rot=128, layout="pairs",
             norm=False, x="f32", cache="f32"),
        # one decoded token of the smallest decoder behind 700 positions
        dict(name="paged_token_700", kind="attention", S=1, T=1, NH=14, NKV=2, HD=64, P=16, least=700, most=700, x="f32", cache="f16"),
        # a decode step of 64 sequences of 50 to 8000 positions
        dict(name="paged_batch64_8000", kind="attention", S=64, T=1, NH=32, NKV=8, HD=128, P=64, least=50, most=8000, x="f16", cache="f16"),
        # one token at the end of a long context
        dict(name="paged_token_131000", kind="attention", S=1, T=1, NH=32, NKV=8, HD=128, P=256, least=131000, most=131000, x="f32",
             cache="f16"),
        # up to 4 drafted tokens and the one before them, of 16 sequences, fp32 cache
        dict(name="paged_drafts16_5", kind="attention", S=16, T=5, NH=28, NKV=4, HD=128, P=32, least=300, most=5000, x="f32", cache="f32"),
        # 4 drafted tokens of one sequence
        dict(name="verify_1x4", kind="verify", S=1, D=4, V=151936, draft=True, temperature=1.0, masked=0.0, x="f32"),
        # 4 drafted tokens of 64 sequences
        dict(name="verify_64x4", kind="verify", S=64, D=4, V=128256, draft=True, temperature=0.8, masked=0.0, x="f32"),
        # 6 tokens looked up in the text, of 24 sequences, a third of the vocabulary masked (constrained decoding)
        dict(name="verify_24x6_lookup", kind="verify", S=24, D=6, V=32003, draft=False, temperature=0.7, masked=0.33, x="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "attention", "attention", "verify"])
    x = rng.choice(["f32", "f16"])
    NH, NKV, HD = rng.choice(HEADS)
    layout = rng.choice(["half", "pairs"])
    rot = rng.choice([HD, HD, HD // 2, HD // 4])
    if kind == "rope":
        return dict(kind=kind, T=_log(rng, 1, 220000 // NH), H=NH, HD=HD, rot=rot, layout=layout, scale=rng.choice(["none", "linear", "yarn"]),
                    ctx=rng.choice([8192, 32768, 131072]), x=x, transpose=rng.random() < 0.4, pad=rng.choice([0, 2 * NKV * HD, rng.randint(1, 99)]))
    if kind == "append":
        S = _log(rng, 1, 200)
        return dict(kind=kind, S=S, T=_log(rng, 1, max(1, 5000 // S)), NH=NH, NKV=NKV, HD=HD, P=rng.choice(PAGES),
                    most=rng.choice([0, _log(rng, 1, max(2, min(2000, 20000 // S)))]), rot=rot, layout=layout, norm=rng.random() < 0.5, x=x,
                    cache=rng.choice(["f16", "f32"]))
    if kind == "attention":
        S = _log(rng, 1, 128)
        T = rng.choice([1, 1, rng.randint(2, 9)])
        most = _log(rng, 10, 220000 // S)
        return dict(kind=kind, S=S, T=T, NH=NH, NKV=NKV, HD=HD, P=rng.choice(PAGES), least=rng.choice([1, most]), most=most, x=x,
                    cache=rng.choice(["f16", "f16", "f32"]))
    S, D, V = _log(rng, 1, 60), rng.randint(0, 6), rng.choice([151936, 128256, rng.randint(1000, 150000)])
    draft = rng.random() < 0.6
    S = max(1, min(S, 60000000 // (V * (2 * D + 1))))
    return dict(kind=kind, S=S, D=D, V=V, draft=draft, temperature=rng.choice([0.0, 0.7, 1.0, rng.uniform(0.3, 1.3)]),
                masked=rng.choice([0.0, 0.0, rng.uniform(0.05, 0.95)]), x=x)


# ---- inputs ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000003 + 41)
    return g


def _dtype(s):
    return torch.float16 if s == "f16" else torch.float32


def _heads(g, n, HD, rows):
    """(rows, n, HD) values N(0, 1) with one channel in 32 of each head four times as large, as keys have."""
    big = 1.0 + 3.0 * (torch.rand((n, HD), device=DEV, generator=g) < 1 / 32).float()
    return torch.randn((rows, n, HD), device=DEV, generator=g) * big


def _tables(rot, n, scale="none"):
    """cos and sin (n, rot / 2), rounded once from float64: plain, every angle a quarter ("linear"), or a ramp
    from the plain angles of the fast pairs to a quarter of the slow ones', times 0.1 ln 4 + 1 ("yarn")."""
    f = 1e6 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    m = 1.0
    if scale == "linear":
        f = f / 4.0
    elif scale == "yarn":
        at = [rot * math.log(n / 4.0 / (b * 2.0 * math.pi)) / (2.0 * math.log(1e6)) for b in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        slow = ((torch.arange(rot // 2, device=DEV, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        f = f * (1.0 - slow) + f / 4.0 * slow
        m = 0.1 * math.log(4.0) + 1.0
    a = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * f[None, :]
    return (a.cos() * m).float(), (a.sin() * m).float()


def _page_table(g, need, most, P):
    """pages (S, pages of `most` positions) of sequences that need[s] positions, in no order, and how many pages the cache has."""
    n = (need + P - 1) // P
    wide = (most + P - 1) // P
    total = need.numel() * wide + 2
    order = torch.randperm(total, device=DEV, generator=g)
    at = torch.arange(wide, device=DEV)[None, :]
    table = order[((n.cumsum(0) - n)[:, None] + at).clamp(max=total - 1)]
    return torch.where(at < n[:, None], table, -1).to(torch.int32).contiguous(), total


def prepare(case, seed):
    c, g = case, _gen(seed)
    ri = lambda lo, hi, n: torch.randint(lo, hi + 1, (n,), device=DEV, generator=g)  # noqa: E731
    if c["kind"] == "rope":
        T, H, HD = c["T"], c["H"], c["HD"]
        x = torch.cat([_heads(g, H, HD, T).reshape(T, -1), torch.randn((T, c["pad"]), device=DEV, generator=g)], 1).to(_dtype(c["x"]))
        first = int(ri(0, c["ctx"] - T, 1)) if T < c["ctx"] else 0
        pos = first + torch.arange(T, device=DEV) if T > 512 else ri(0, c["ctx"] - 1, T)
        cos, sin = _tables(c["rot"], c["ctx"], c["scale"])
        return {"case": c, "x": x[:, :H * HD].unflatten(1, (H, HD)), "positions": pos.clamp(max=c["ctx"] - 1).to(torch.int32), "cos": cos, "sin": sin}
    if c["kind"] == "verify":
        S, D, V, t = c["S"], c["D"], c["V"], _dtype(c["x"])
        # rows from flat to peaked, as positions of a text are; the draft's are the target's with an error
        x = torch.randn((S, D + 1, V), device=DEV, generator=g) * (1.5 + 2.0 * torch.rand((S, D + 1, 1), device=DEV, generator=g))
        d = (x[:, :D] + 0.7 * torch.randn((S, D, V), device=DEV, generator=g)).to(t)
        if c["masked"]:
            x[:, :, torch.rand(V, device=DEV, generator=g) < c["masked"]] = -math.inf
        tau = c["temperature"] or 1e-3
        drafts = torch.empty((S, D), dtype=torch.int32, device=DEV)
        for i in range(D):  # drawn from the draft's distribution, with exponential noise
            e = torch.empty((S, V), device=DEV).exponential_(generator=g)
            drafts[:, i] = (d[:, i].float() / tau - e.log()).argmax(1).to(torch.int32)
        if not c["draft"] or c["temperature"] == 0:  # most tokens looked up, and most of a greedy draft, are likely ones
            likely = torch.rand((S, D, 1), device=DEV, generator=g) < 0.7
            x[:, :D].scatter_add_(2, drafts.long()[:, :, None], torch.where(likely, 12.0, 0.0))
        short = torch.rand(S, device=DEV, generator=g) < 0.2  # some sequences have fewer drafts
        few = ri(0, max(D - 1, 0), S)
        drafts[short[:, None] & (torch.arange(D, device=DEV)[None, :] >= few[:, None])] = -1
        return {"case": c, "logits": x.to(t), "draft_logits": d if c["draft"] else None, "drafts": drafts,
                "uniforms": torch.rand((S, D + 1), device=DEV, generator=g)}
    S, T, NH, NKV, HD, P = c["S"], c["T"], c["NH"], c["NKV"], c["HD"], c["P"]
    if c["kind"] == "append":
        before = ri(0, c["most"], S) if c["most"] else torch.zeros(S, dtype=torch.int64, device=DEV)
        new = ri((T + 4) // 5, T, S)  # tokens of each sequence: a padded batch
        new[0] = T
    else:
        new = ri((T + 1) // 2, T, S)
        new[0] = T
        before = (ri(c["least"], c["most"], S) - new).clamp(min=0)
        before[0] = max(c["most"] - T, 0)
    at = torch.arange(T, device=DEV)[None, :]
    pos = torch.where(at < new[:, None], before[:, None] + at, -1).to(torch.int32)
    pages, total = _page_table(g, before + new, max(c["most"], T) if c["kind"] == "attention" else c["most"] + T, P)
    st = {"case": c, "positions": pos, "pages": pages}
    if c["kind"] == "attention":
        n = total * P
        k, v = _heads(g, NKV, HD, n).to(_dtype(c["cache"])), torch.randn((n, NKV, HD), device=DEV, generator=g).to(_dtype(c["cache"]))
        st["cache"] = torch.stack([t.reshape(total, P, NKV, HD).transpose(1, 2) for t in (k, v)], 1).contiguous()
        st["q"] = torch.randn((S, T, NH, HD), device=DEV, generator=g).to(_dtype(c["x"]))
        return st
    qkv = torch.cat([_heads(g, NH, HD, S * T), _heads(g, NKV, HD, S * T), torch.randn((S * T, NKV, HD), device=DEV, generator=g)], 1)
    st["qkv"] = qkv.reshape(S, T, -1).to(_dtype(c["x"]))
    st["cos"], st["sin"] = _tables(c["rot"], c["most"] + T)
    st["qn"], st["kn"] = ((1.0 + 0.2 * torch.randn(HD, device=DEV, generator=g) for _ in range(2)) if c["norm"] else (None, None))
    st["cache"] = torch.zeros((total, 2, NKV, P, HD), dtype=_dtype(c["cache"]), device=DEV)
    return st


# ---- one pass -------------------------------------------------------------------------
def _rotate(x, cos, sin, pairs):
    """x (.., HD) fp32, its first 2 R dimensions rotated by cos and sin (.., R)."""
    R = cos.shape[-1]
    a, b = (x[..., 0:2 * R:2], x[..., 1:2 * R:2]) if pairs else (x[..., :R], x[..., R:2 * R])
    u, w = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([u, w], -1).flatten(-2) if pairs else torch.cat([u, w], -1)
    return torch.cat([y, x[..., 2 * R:]], -1)


def _run_rope(s):
    c = s["case"]
    if own:
        from webpytorch_amd import core
        return core.rope(s["x"], s["positions"], core.Rope(s["cos"], s["sin"], c["layout"] == "pairs"), transpose=c["transpose"])
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    return _rotate(s["x"].float(), cos, -sin if c["transpose"] else sin, c["layout"] == "pairs").to(s["x"].dtype)


def _run_append(s):
    c = s["case"]
    S, T, NH, NKV, HD, P = c["S"], c["T"], c["NH"], c["NKV"], c["HD"], c["P"]
    pairs = c["layout"] == "pairs"
    if own:
        from webpytorch_amd import core
        q = core.paged_append(s["qkv"], s["positions"], s["pages"], s["cache"], NH, core.Rope(s["cos"], s["sin"], pairs), qn=s["qn"], kn=s["kn"])
        return {"q": q, "cache": s["cache"]}
    pos = s["positions"].long()
    there = pos >= 0
    at = pos.clamp(min=0)
    x = s["qkv"].float().reshape(S, T, NH + 2 * NKV, HD)
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    q, k, v = x[:, :, :NH], x[:, :, NH:NH + NKV], x[:, :, NH + NKV:]
    if s["qn"] is not None:
        q, k = (t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w for t, w in ((q, s["qn"]), (k, s["kn"])))
    q = _rotate(q, cos, sin, pairs) * there[:, :, None, None]
    k = _rotate(k, cos, sin, pairs)
    page, slot = s["pages"].long().gather(1, at // P)[there], (at % P)[there]
    s["cache"][page, 0, :, slot] = k[there].to(s["cache"].dtype)
    s["cache"][page, 1, :, slot] = v[there].to(s["cache"].dtype)
    return {"q": q.to(s["qkv"].dtype), "cache": s["cache"]}


def _run_attention(s):
    c = s["case"]
    if own:
        from webpytorch_amd import core
        return core.paged_attention(s["q"], s["positions"], s["pages"], s["cache"])
    S, T, NH, NKV, HD = c["S"], c["T"], c["NH"], c["NKV"], c["HD"]
    rep = NH // NKV
    kv = s["cache"][s["pages"].long().clamp(min=0)]  # (S, pages, 2, NKV, P, HD)
    k, v = (kv[:, :, i].transpose(1, 2).flatten(2, 3).float() for i in range(2))
    n = k.shape[2]
    q = s["q"].float().reshape(S, T, NKV, rep, HD).permute(0, 2, 3, 1, 4).reshape(S, NKV, rep * T, HD)
    a = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(HD)).reshape(S, NKV, rep, T, n)
    later = torch.arange(n, device=DEV)[None, None, :] > s["positions"][:, :, None]
    a.masked_fill_(later[:, None, None], -math.inf)
    m = a.amax(-1, keepdim=True)
    a = (a - torch.where(m == -math.inf, 0.0, m)).exp_()
    z = a.sum(-1, keepdim=True)
    a = a / torch.where(z == 0, 1.0, z)
    o = torch.matmul(a.reshape(S, NKV, rep * T, n), v)
    return o.reshape(S, NKV, rep, T, HD).permute(0, 3, 1, 2, 4).reshape(S, T, NH, HD).to(s["q"].dtype)


def _run_verify(s):
    """Probabilities and running sums in float64: a draw has to fall on the same side of every border."""
    c = s["case"]
    S, D = c["S"], c["D"]
    if own:
        from webpytorch_amd import core
        r = core.verify_drafts(s["logits"], s["drafts"], s["uniforms"], s["draft_logits"], temperature=c["temperature"])
        return {"tokens": r.tokens, "accepted": r.accepted}
    x, ids = s["logits"].double(), s["drafts"].long()
    tau = c["temperature"]
    at = ids.clamp(min=0)[:, :, None]
    if tau > 0:
        p = torch.exp((x - x.amax(-1, keepdim=True)) / tau)
        p = p / p.sum(-1, keepdim=True)
    else:
        p = torch.zeros_like(x).scatter_(2, x.argmax(-1, keepdim=True), 1.0)
    if tau > 0 and s["draft_logits"] is not None:
        d = s["draft_logits"].double()
        q = torch.exp((d - d.amax(-1, keepdim=True)) / tau)
        q = q / q.sum(-1, keepdim=True)
    else:
        q = torch.zeros_like(x[:, :D]).scatter_(2, at, 1.0)
    u = s["uniforms"].double()
    ok = (ids >= 0) & (u[:, :D] * q.gather(2, at)[:, :, 0] < p[:, :D].gather(2, at)[:, :, 0])
    n = ok.long().cumprod(1).sum(1)  # accepted
    row = torch.arange(S, device=DEV)
    w = p[row, n]
    if D:
        inside = n.clamp(max=D - 1)
        rejected = (n < D) & (ids[row, inside] >= 0)
        w = torch.where(rejected[:, None], (w - q[row, inside]).clamp(min=0.0), w)
    run_sum = w.cumsum(1)
    token = ((run_sum > u[:, D:] * run_sum[:, -1:]) & (w > 0)).to(torch.uint8).argmax(1)
    tokens = torch.cat([torch.where(torch.arange(D, device=DEV)[None, :] < n[:, None], ids, -1), torch.full((S, 1), -1, device=DEV)], 1)
    tokens[row, n] = token
    return {"tokens": tokens.to(torch.int32), "accepted": n.to(torch.int32)}


def run(state):
    return {"rope": _run_rope, "append": _run_append, "attention": _run_attention, "verify": _run_verify}[state["case"]["kind"]](state)


def work(case):
    c = case
    size = 2 if c["x"] == "f16" else 4
    if c["kind"] == "rope":
        return {"bytes": 2 * c["T"] * c["H"] * c["HD"] * size + c["T"] * c["rot"] * 4, "flops": 3 * c["T"] * c["H"] * c["rot"]}
    if c["kind"] == "verify":
        n = c["S"] * (c["D"] * (2 if c["draft"] and c["temperature"] > 0 else 1) + 1) * c["V"]
        return {"bytes": n * size + c["S"] * (3 * c["D"] + 3) * 4, "flops": 4 * n}
    S, T, NH, NKV, HD = c["S"], c["T"], c["NH"], c["NKV"], c["HD"]
    wide = 2 if c["cache"] == "f16" else 4
    if c["kind"] == "append":
        rows = S * (0.6 * T if T > 1 else 1)  # a padded batch is three fifths full
        return {"bytes": rows * (((2 * NH + 2 * NKV) * size + 2 * NKV * wide) * HD + c["rot"] * 4), "flops": rows * (NH + NKV) * HD * 7}
    keys = S * (c["least"] + c["most"]) / 2
    return {"bytes": keys * 2 * NKV * HD * wide + 2 * S * T * NH * HD * size, "flops": 4 * NH * HD * keys * T}


# ---- the same in float64 ----------------------------------------------------------------
def _turn(x, cos, sin, pairs):
    """x (.., HD) float64 as complex numbers times cos + i sin."""
    R = cos.shape[-1]
    head = x[..., :2 * R]
    z = head.unflatten(-1, (R, 2)) if pairs else head.unflatten(-1, (2, R)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * torch.complex(cos, sin))
    z = z.flatten(-2) if pairs else z.transpose(-1, -2).flatten(-2)
    return torch.cat([z, x[..., 2 * R:]], -1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "rope":
        cos, sin = (t[s["positions"].long()].double()[:, None] for t in (s["cos"], s["sin"]))
        return _turn(s["x"].double(), cos, -sin if c["transpose"] else sin, c["layout"] == "pairs")
    if c["kind"] == "verify":
        tokens = torch.full((c["S"], c["D"] + 1), -1, dtype=torch.int32)
        accepted = torch.zeros(c["S"], dtype=torch.int32)
        tau, V = c["temperature"], c["V"]

        def law(row):
            if tau == 0:
                return torch.nn.functional.one_hot(torch.argmax(row), V).double()
            return torch.softmax(row.double() / tau, 0)
        for b in range(c["S"]):
            u, i = s["uniforms"][b].double(), 0
            while True:
                weights = law(s["logits"][b, i])
                x = int(s["drafts"][b, i]) if i < c["D"] else -1
                if x < 0:
                    break
                given = law(s["draft_logits"][b, i]) if s["draft_logits"] is not None and tau > 0 else \
                    torch.nn.functional.one_hot(torch.tensor(x, device=DEV), V).double()
                if not float(u[i] * given[x]) < float(weights[x]):
                    weights = torch.relu(weights - given)
                    break
                tokens[b, i] = x
                i += 1
            total = torch.cumsum(weights, 0)
            tokens[b, i] = int(torch.searchsorted(total, (u[-1] * total[-1]).reshape(1), right=True))
            accepted[b] = i
        return {"tokens": tokens.to(DEV), "accepted": accepted.to(DEV)}
    S, T, NH, NKV, HD, P = c["S"], c["T"], c["NH"], c["NKV"], c["HD"], c["P"]
    if c["kind"] == "attention":
        out = torch.zeros((S, T, NH, HD), dtype=torch.float64, device=DEV)
        for b in range(S):
            pos = s["positions"][b].long()
            n = int(pos.max()) + 1
            at = torch.arange(n, device=DEV)
            rows = s["cache"][s["pages"][b].long()[at // P], :, :, at % P]  # (n, 2, NKV, HD)
            gone = at[None, :] > pos[:, None]
            for h in range(NH):
                k, v = (rows[:, i, h // (NH // NKV)].double() for i in range(2))
                a = torch.mm(s["q"][b, :, h].double(), k.t().contiguous()) / math.sqrt(HD)
                a[gone] = -math.inf
                out[b, :, h] = torch.mm(torch.nan_to_num(torch.softmax(a, 1), nan=0.0), v)
        return out
    keep = s["positions"] >= 0
    pos = s["positions"].long() * keep
    cos, sin = (t.double()[pos][:, :, None] for t in (s["cos"], s["sin"]))
    parts = list(s["qkv"].double().unflatten(-1, (NH + 2 * NKV, HD)).split([NH, NKV, NKV], 2))
    for i, w in enumerate((s["qn"], s["kn"])):
        if w is not None:
            parts[i] = parts[i] * torch.rsqrt(parts[i].pow(2).sum(-1, keepdim=True) / HD + 1e-6) * w.double()
        parts[i] = _turn(parts[i], cos, sin, c["layout"] == "pairs")
    full = s["cache"].double()
    for b, t in keep.nonzero().tolist() if S * T <= 400 else ():
        full[int(s["pages"][b, pos[b, t] // P]), :, :, int(pos[b, t]) % P] = torch.stack([parts[1][b, t], parts[2][b, t]])
    if S * T > 400:  # the same by flat slots: (page, which, head, slot)
        page = torch.take_along_dim(s["pages"].long(), pos // P, 1)
        which, head = torch.arange(2, device=DEV)[:, None], torch.arange(NKV, device=DEV)[None, :]
        flat = ((page[..., None, None] * 2 + which) * NKV + head) * P + (pos % P)[..., None, None]
        rows = torch.stack([parts[1], parts[2]], 2)
        full.view(-1, HD).index_copy_(0, flat[keep].reshape(-1), rows[keep].reshape(-1, HD))
    return {"q": parts[0] * keep[:, :, None, None], "cache": full}
