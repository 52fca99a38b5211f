"""GPU: QK-norm + RoPE + cache write, the 4-bit cache and attention over it, against float64
(`oracle/kv4.py`)."""
import math
import threading

import numpy as np
import pytest

from oracle import kv4

pytestmark = pytest.mark.gpu

F32_REL = 5e-6  # q and p carry 22 bits (2^-22 each, scores of a few units), fp32 sums the rest
# fp16 rows: the output's rounding (2^-12 of a value on average, 2^-11 at most) and p's, as large
F16_REL = 2.0 ** -11


def tables(torch, n, hd):
    ang = np.arange(n, dtype=np.float64)[:, None] / (1e6 ** (np.arange(0, hd, 2, dtype=np.float64) / hd))
    return torch.from_numpy(np.cos(ang).astype(np.float32)).cuda(), torch.from_numpy(np.sin(ang).astype(np.float32)).cuda()


def state(torch, pos):
    return torch.tensor([pos, 0, 0, 0], dtype=torch.int32, device="cuda")


def fill(k, v, start=0, cache=None, lmax=None):
    """k and v (n, NKV, HD) torch fp32 written to positions start .. through the operator, unrotated."""
    import torch
    from webpytorch_amd import core
    n, nkv, hd = k.shape
    lmax = lmax or start + n
    cache = core.kv4_cache(nkv, lmax, hd) if cache is None else cache
    qkv = torch.cat([torch.zeros((n, nkv, hd)), k, v], 1).reshape(n, -1).cuda()
    rows = cache.shape[1] * 32
    core.qk_norm_rope(qkv, state(torch, start), torch.ones((rows, hd // 2), device="cuda"), torch.zeros((rows, hd // 2), device="cuda"),
                      nkv, cache)
    return cache


def close(got, want, rel):
    got = got.double().cpu().numpy()
    assert got.shape == want.shape and np.isfinite(got).all()
    norm = np.linalg.norm(want)
    assert np.linalg.norm(got - want) <= rel * norm + 1e-30, np.linalg.norm(got - want) / norm
    assert np.abs(got - want).max() <= 20 * rel * max(norm / math.sqrt(want.size), np.abs(want).max())


# ---- QK-norm + RoPE + cache write ----
@pytest.mark.parametrize("NH,NKV,HD", [(14, 2, 64), (4, 4, 32), (3, 1, 80), (6, 2, 96), (8, 2, 128), (2, 1, 256), (5, 5, 2)])
@pytest.mark.parametrize("T,pos,norm", [(1, 0, "qk"), (1, 39, "q"), (7, 3, "k"), (9, 31, ""), (33, 7, "qk")])
def test_fp32_cache_is_the_two_calls_bit_for_bit(gpu, NH, NKV, HD, T, pos, norm):
    import torch
    from webpytorch_amd import _lib, core
    g = torch.Generator().manual_seed(T + HD)
    W, LMAX = (NH + 2 * NKV) * HD, 40
    padded = torch.randn((T, W + 5), generator=g).cuda()
    qkv = padded[:, :W]
    qn, kn = (torch.randn(HD, generator=g).cuda() if c in norm else None for c in "qk")
    cos, sin = tables(torch, LMAX, HD)
    st = state(torch, pos)
    a, b = ([torch.full((NKV, LMAX, HD), 3.0, device="cuda") for _ in range(2)] for _ in range(2))
    got = core.qk_norm_rope(qkv, st, cos, sin, NH, a, qn=qn, kn=kn, eps=1e-5)
    x, q = qkv.clone().contiguous(), torch.zeros((T, NH, HD), device="cuda")
    P = core.ptr
    if norm:
        _lib.call("miq_head_rmsnorm", P(x), P(qn), P(kn), T, NH, NKV, HD, 1e-5, None)
    _lib.call("miq_rope_kv", P(x), P(st), P(cos), P(sin), P(q), P(b[0]), P(b[1]), T, NH, NKV, HD, LMAX, None)
    assert torch.equal(got, q) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dt", ["float32", "float16"])
@pytest.mark.parametrize("NH,NKV,HD", [(14, 2, 64), (8, 2, 128), (2, 1, 192), (4, 1, 256)])
@pytest.mark.parametrize("T,pos,norm", [(1, 0, "qk"), (1, 45, ""), (3, 30, "k"), (32, 32, "q"), (70, 13, "qk")])
def test_kv4_write_matches_float64(gpu, NH, NKV, HD, T, pos, norm, dt):
    """q to a rounding of its type; the codes, S and Z equal; the other positions' as they were."""
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(T * 7 + HD)
    lmax = 96
    qkv = (torch.randn((T, (NH + 2 * NKV) * HD), generator=g) * 2).to(getattr(torch, dt))
    qn, kn = (1 + 0.3 * torch.randn(HD, generator=g) if c in norm else None for c in "qk")
    before = torch.randint(0, 256, (NKV, 3, 40 * HD), dtype=torch.uint8, generator=g)
    cache = before.cuda()
    cos, sin = tables(torch, lmax, HD)
    q = core.qk_norm_rope(qkv.cuda(), state(torch, pos), cos, sin, NH, cache, qn=None if qn is None else qn.cuda(),
                          kn=None if kn is None else kn.cuda())
    x = qkv.float().numpy().reshape(T, -1, HD)
    c, s = (t[pos:pos + T].cpu().numpy() for t in (cos, sin))
    wq = kv4.norm_rope(x[:, :NH], None if qn is None else qn.numpy(), c, s)
    wk = kv4.norm_rope(x[:, NH:NH + NKV], None if kn is None else kn.numpy(), c, s).astype(np.float32)
    assert q.dtype == qkv.dtype
    ulp = 2.0 ** (-24 if dt == "float32" else -11)
    assert (np.abs(q.double().cpu().numpy() - wq) <= ulp * np.abs(wq) * 1.001 + 2.0 ** -24).all()
    was, now = kv4.unpack(before.numpy(), lmax), kv4.unpack(cache.cpu().numpy(), lmax)
    at = np.arange(pos, pos + T)
    rest = np.setdiff1d(np.arange(lmax), at)
    for part, rows in ((0, wk), (1, x[:, NH + NKV:])):
        want = kv4.quantize(np.ascontiguousarray(rows.transpose(1, 0, 2)))
        for i in range(3):
            assert np.array_equal(now[part][i][:, at], want[i], equal_nan=i > 0)
            view = (lambda t: t) if i == 0 else (lambda t: np.ascontiguousarray(t).view(np.uint16))
            assert np.array_equal(view(now[part][i])[:, rest], view(was[part][i])[:, rest])


def test_kv4_groups_of_every_kind(gpu):
    """Constant, tiny, saturating, offset and non-finite groups, read back."""
    import torch
    from webpytorch_amd import core
    rng = np.random.default_rng(5)
    x = rng.standard_normal((12, 1, 64)).astype(np.float32)
    x[1], x[2], x[3] = 0, 1.25, x[3] * 1e-8
    x[4], x[5] = x[4] * 1e5, 100 + x[5] * 1e-3
    x[6, 0, 3], x[7, 0, 40], x[8, 0, 63] = np.nan, np.inf, -np.inf
    x[9], x[10] = -16384, np.where(np.arange(64) % 2, 16384, -16384)
    k, v = torch.from_numpy(x), torch.from_numpy(x[::-1].copy())
    cache = fill(k, v)
    gk, gv = core.kv4_dequant(cache, 0, 12)
    turned = kv4.norm_rope(x, None, np.ones((12, 32)), np.zeros((12, 32))).astype(np.float32)  # 0 times a NaN is one
    for got, src in ((gk, turned), (gv, x[::-1])):
        want = kv4.stands_for(*kv4.quantize(np.ascontiguousarray(src.transpose(1, 0, 2))))
        assert np.array_equal(got.cpu().numpy(), want, equal_nan=True)
    part = core.kv4_dequant(cache, 5, 3)
    assert torch.equal(part[1].nan_to_num(7.0), gv[:, 5:8].nan_to_num(7.0)) and torch.equal(part[0].nan_to_num(7.0), gk[:, 5:8].nan_to_num(7.0))


@pytest.mark.parametrize("four", [True, False])
@pytest.mark.parametrize("pos", [-3, 62, 64, 2 ** 31 - 2])
def test_positions_outside_the_cache(gpu, four, pos):
    import torch
    from webpytorch_amd import core
    T, NH, NKV, HD, n = 5, 4, 2, 64, 64
    qkv = torch.randn((T, (NH + 2 * NKV) * HD), generator=torch.Generator().manual_seed(1)).cuda()
    cos, sin = tables(torch, n, HD)
    new = lambda: core.kv4_cache(NKV, n, HD) if four else [torch.zeros((NKV, n, HD), device="cuda") for _ in range(2)]  # noqa: E731
    cache, ref = new(), new()
    q = core.qk_norm_rope(qkv, state(torch, pos), cos, sin, NH, cache, out=torch.full((T, NH, HD), 7.0, device="cuda"))
    inside = [t for t in range(T) if 0 <= pos + t < n]
    for t in range(T):
        if t in inside:  # one by one into another cache
            one = core.qk_norm_rope(qkv[t:t + 1], state(torch, pos + t), cos, sin, NH, ref)
            assert torch.equal(q[t:t + 1], one)
        else:
            assert not q[t].any()
    pairs = [(cache, ref)] if four else list(zip(cache, ref))
    assert all(torch.equal(a, b) for a, b in pairs)


# ---- attention ----
HEADS = [(14, 2, 64), (3, 1, 128), (8, 8, 64), (2, 1, 192), (4, 1, 256), (16, 2, 128), (40, 2, 64)]


@pytest.mark.parametrize("dt", ["float32", "float16"])
@pytest.mark.parametrize("NH,NKV,HD", HEADS)
@pytest.mark.parametrize("T,pos,lmax", [(1, 0, 1), (1, 31, 64), (1, 700, 2048), (2, 255, 257), (17, 0, 40), (33, 127, 160), (5, 500, 505),
                                        (130, 3, 140), (96, 300, 4096)])
def test_attention_matches_float64(gpu, NH, NKV, HD, T, pos, lmax, dt):
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(T * 1000 + pos + HD)
    n = pos + T
    q = torch.randn((T, NH, HD), generator=g).to(getattr(torch, dt))
    k, v = (torch.randn((n, NKV, HD), generator=g) for _ in range(2))
    cache = fill(k, v, lmax=lmax)
    got = core.attention_kv4(q.cuda(), cache, state(torch, pos))
    assert got.dtype == q.dtype
    wk, wv = (t.cpu().numpy() for t in core.kv4_dequant(cache, 0, n))
    close(got, kv4.attention(q.float().numpy(), wk, wv, pos, 1 / math.sqrt(HD)), F32_REL if dt == "float32" else F16_REL)


@pytest.mark.parametrize("scale,size", [(1.0, 1e-30), (1e-3, 1e30), (0.125, 60000.0), (3.0, 1.0), (0.0, 1.0), (-0.2, 1.0)])
def test_query_magnitudes_and_scales(gpu, scale, size):
    """Queries far from 1 are scaled by a power of two, so nothing leaves fp16's range; scores stay moderate or
    pick one key."""
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(3)
    T, NH, NKV, HD, pos = 3, 4, 2, 64, 90
    q = torch.randn((T, NH, HD), generator=g) * size
    k, v = (torch.randn((pos + T, NKV, HD), generator=g) for _ in range(2))
    cache = fill(k, v)
    s = scale / max(size, 1e-20) if size != 1.0 else scale
    got = core.attention_kv4(q.cuda(), cache, state(torch, pos), scale=s)
    wk, wv = (t.cpu().numpy() for t in core.kv4_dequant(cache, 0, pos + T))
    s = float(np.float32(s))
    want = kv4.attention(q.numpy(), wk, wv, pos, s)
    # scores reach |s| = 3 x 8 x 8 at the steepest: their 2^-22 is that much of p
    close(got, want, 5e-5 if abs(scale) > 1 else F32_REL)


@pytest.mark.parametrize("NH,NKV,HD,T", [(4, 2, 64, 40), (2, 1, 128, 40), (14, 2, 64, 1), (8, 1, 128, 200)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_non_finite_rows_reach_only_their_queries(gpu, NH, NKV, HD, T, which):
    """A NaN in a group of position 20, and memory of any kind behind the last position: tokens before position
    20 are what they are without it."""
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(HD)
    pos = 30 if T == 1 else 5
    lmax = T + 70
    q = torch.randn((T, NH, HD), generator=g).cuda()
    k, v = (torch.randn((T + pos, NKV, HD), generator=g) for _ in range(2))
    rnd = torch.randint(0, 256, (NKV, (lmax + 31) // 32, 40 * HD), dtype=torch.uint8, generator=g)
    clean, dirty = fill(k, v, lmax=lmax), fill(k, v, cache=rnd.cuda())
    a, b = (core.attention_kv4(q, c, state(torch, pos)) for c in (clean, dirty))
    assert torch.isfinite(a).all() and torch.equal(a, b)
    (k if which == "k" else v)[20, 0, 37] = float("nan")
    got = core.attention_kv4(q, fill(k, v, cache=rnd.cuda()), state(torch, pos))
    sees = torch.arange(T) + pos >= 20
    assert torch.equal(got[~sees], a[~sees])
    of = torch.arange(NH) < NH // NKV  # the heads of kv head 0
    assert torch.equal(got[sees][:, ~of], a[sees][:, ~of])
    hit = got[sees][:, of]
    if which == "k":
        assert torch.isnan(hit).all()
    else:
        assert torch.isnan(hit[..., 32:64]).all()
        other = [d for d in range(HD) if not 32 <= d < 64]
        assert torch.equal(hit[..., other], a[sees][:, of][..., other])


def test_tokens_without_a_key_are_zero(gpu):
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(9)
    T, NH, NKV, HD = 9, 6, 2, 64
    q = torch.randn((T, NH, HD), generator=g)
    k, v = (torch.randn((32, NKV, HD), generator=g) for _ in range(2))
    cache = fill(k, v)
    wk, wv = (t.cpu().numpy() for t in core.kv4_dequant(cache))
    for pos in (-4, -100, -2 ** 31):
        got = core.attention_kv4(q.cuda(), cache, state(torch, pos))
        close(got, kv4.attention(q.numpy(), wk, wv, pos, 1 / 8), F32_REL)
        assert not got[:min(T, -pos)].any()
    got = core.attention_kv4(q.cuda(), cache, state(torch, 28))  # past the cache's end: its last key
    close(got, kv4.attention(q.numpy(), wk, wv, 28, 1 / 8), F32_REL)


def test_values_of_the_largest_size(gpu):
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(11)
    n, HD = 3000, 64
    q = torch.randn((1, 4, HD), generator=g) * 0.01
    k, v = torch.randn((n, 1, HD), generator=g), torch.rand((n, 1, HD), generator=g) * 8000 + 8000
    cache = fill(k, v)
    wk, wv = (t.cpu().numpy() for t in core.kv4_dequant(cache, 0, n))
    close(core.attention_kv4(q.cuda(), cache, state(torch, n - 1)), kv4.attention(q.numpy(), wk, wv, n - 1, 1 / 8), F32_REL)


def test_cache_past_4_gib(gpu):
    """Records of the last kv head lie past 2^32 bytes: keys of zero, so that every position counts alike, and
    values in the last 40 positions only."""
    import torch
    from webpytorch_amd import core
    NKV, HD, n = 8, 128, 3_500_000
    cache = core.kv4_cache(NKV, n, HD)
    assert cache.numel() > 4 << 30
    g = torch.Generator().manual_seed(2)
    v = torch.randn((40, NKV, HD), generator=g)
    qkv = torch.cat([torch.zeros((40, 2 * NKV, HD)), v], 1).reshape(40, -1).cuda()
    one, zero = torch.ones((cache.shape[1] * 32, HD // 2), device="cuda"), torch.zeros((cache.shape[1] * 32, HD // 2), device="cuda")
    core.qk_norm_rope(qkv, state(torch, n - 40), one, zero, NKV, cache)
    wv = core.kv4_dequant(cache, n - 40, 40)[1].cpu().double().numpy()
    for T in (1, 20):
        q = torch.randn((T, NKV, HD), generator=g)
        got = core.attention_kv4(q.cuda(), cache, state(torch, n - T))
        want = np.stack([wv[:, :40 - T + 1 + t].sum(1) / (n - T + 1 + t) for t in range(T)])
        close(got, want, F32_REL)


# ---- streams, graphs, threads ----
def _case(seed, T=1, NH=8, NKV=2, HD=64, pos=1500, lmax=4096):
    import torch
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((pos + T, NKV, HD), generator=g) for _ in range(2))
    q = torch.randn((T, NH, HD), generator=g).cuda()
    return q, fill(k, v, lmax=lmax), state(torch, pos)


def test_attention_is_deterministic_and_leaves_its_workspace_ready(gpu):
    import torch
    from webpytorch_amd import core
    q, cache, st = _case(1)
    first = core.attention_kv4(q, cache, st)
    for T in (1, 30, 1, 3):
        q2, c2, s2 = _case(2 + T, T=T)
        core.attention_kv4(q2, c2, s2)
        assert torch.equal(core.attention_kv4(q, cache, st), first)


def test_two_graphs_replayed_at_a_time(gpu):
    """Captured calls have workspaces of their own: two graphs on two streams, three replays each with eager
    calls between."""
    import torch
    from webpytorch_amd import core
    cases = [_case(21, lmax=8192, pos=7000), _case(22, lmax=8192, pos=6990)]
    want = [core.attention_kv4(*c) for c in cases]
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(core.attention_kv4(*c))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
        assert torch.equal(core.attention_kv4(*cases[0]), want[0])


def test_two_threads_two_streams(gpu):
    import torch
    from webpytorch_amd import core
    cases = [_case(31, pos=4000), _case(32, T=3, pos=4050)]
    want = [core.attention_kv4(*c) for c in cases]
    torch.cuda.synchronize()
    wrong, errors = [0, 0], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                bad = torch.zeros((), dtype=torch.int64, device="cuda")
                for _ in range(50):
                    bad += (core.attention_kv4(*cases[i]) != want[i]).sum()
                wrong[i] = int(bad)
        except Exception as e:
            errors.append(e)
    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join(60)
    assert not errors and wrong == [0, 0], (errors, wrong)


def _torch_want(q, cache, pos):
    """float64 on the GPU over what the cache stands for; q (T, NH, HD)."""
    import torch
    from webpytorch_amd import core
    T, NH, HD = q.shape
    n = max(pos + T, 1)
    k, v = (t.double() for t in core.kv4_dequant(cache, 0, n))
    rep = NH // k.shape[0]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    later = torch.arange(n, device="cuda")[None, :] > pos + torch.arange(T, device="cuda")[:, None]
    for h in range(NH):
        s = torch.mm(q[:, h].double(), k[h // rep].t().contiguous()) / math.sqrt(HD)
        s[later] = -math.inf
        out[:, h] = torch.mm(torch.softmax(s, 1).nan_to_num(0.0), v[h // rep])
    return out


@pytest.mark.parametrize("dt", ["float32", "float16"])
@pytest.mark.parametrize("NH,NKV,HD", [(2, 1, 64), (3, 1, 128), (2, 2, 192), (4, 1, 256)])
@pytest.mark.parametrize("T,pos,lmax", [(600, 0, 600), (300, 5, 8192), (90, 4001, 70000), (257, 1000, 40000), (700, -650, 800),
                                        (700, -20, 8192)])
def test_many_rows(gpu, NH, NKV, HD, T, pos, lmax, dt):
    """The many-row kernel at every head dimension, whole and in slices that a second launch joins, a cache
    whose memory behind the last position is anything, rows before position 0, and a NaN that reaches its tokens."""
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(T + HD)
    n = max(pos + T, 1)
    q = torch.randn((T, NH, HD), generator=g).to(getattr(torch, dt)).cuda()
    k, v = (torch.randn((n, NKV, HD), generator=g) for _ in range(2))
    rnd = torch.randint(0, 256, (NKV, (lmax + 31) // 32, 40 * HD), dtype=torch.uint8, generator=g).cuda()
    cache = fill(k, v, cache=rnd)
    got = core.attention_kv4(q, cache, state(torch, pos))
    want = _torch_want(q, cache, pos)
    close(got, want.cpu().numpy(), F32_REL if dt == "float32" else F16_REL)
    assert not got[:max(0, -pos)].any()
    at = n - min(T, n) // 2 - 1
    v[at, 0, 40] = float("nan")
    bad = core.attention_kv4(q, fill(k, v, cache=rnd), state(torch, pos))
    sees = torch.arange(T) + pos >= at
    assert torch.equal(bad[~sees], got[~sees]) and torch.isnan(bad[sees][:, :NH // NKV, 32:64]).all()
    other = [d for d in range(HD) if not 32 <= d < 64]
    assert torch.equal(bad[sees][..., other], got[sees][..., other])


def test_threads_on_one_stream_with_other_products(gpu):
    """Attention in two launches, log probabilities and a split GEMV share the stream's workspace: each thread
    gets what it gets alone."""
    import torch
    from webpytorch_amd import core, synth
    q, cache, st = _case(51, T=90, pos=4000, lmax=70000)
    lg, ids = torch.randn((3, 50000), generator=torch.Generator().manual_seed(5)).cuda(), torch.arange(3, dtype=torch.int32, device="cuda")
    L = synth.gptq_layer(5, 4096, 1024, 128, 4)
    lin = core.QuantizedLinear.from_autogptq(L["qweight"], L["qzeros"], L["scales"], None, 128, 4)
    x = torch.from_numpy(synth.activations(5, 3, 4096, np.float32)).cuda()
    calls = [lambda: core.attention_kv4(q, cache, st), lambda: core.token_logprobs(lg, ids, 4).top_logprobs, lambda: lin.forward(x)]
    alone = [c() for c in calls]
    torch.cuda.synchronize()
    wrong, errors, start = [torch.zeros((), dtype=torch.int64, device="cuda") for _ in calls], [], threading.Barrier(len(calls))

    def work(i):
        try:
            start.wait(30)
            for _ in range(100):
                wrong[i] += (calls[i]() != alone[i]).sum()
        except Exception as e:
            errors.append(e)
    ts = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in ts:
        t.start()
    for t in ts:
        t.join(60)
    torch.cuda.synchronize()
    assert not errors and [int(w) for w in wrong] == [0, 0, 0], (errors, wrong)


def test_many_rows_in_a_graph(gpu):
    """Two launches and the graph's own workspace, replayed with eager calls between."""
    import torch
    from webpytorch_amd import core
    q, cache, st = _case(52, T=90, pos=4000, lmax=70000)
    want = core.attention_kv4(q, cache, st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = core.attention_kv4(q, cache, st)
    for pos in (4000, 3900, 4000):
        st[0] = pos
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        eager = core.attention_kv4(q, cache, st)
        assert torch.equal(out, eager) and (pos != 4000 or torch.equal(out, want))


@pytest.mark.parametrize("dt", ["float32", "float16"])
@pytest.mark.parametrize("T", [5, 40, 700])
def test_a_token_does_not_depend_on_its_neighbours(gpu, T, dt):
    """Other tokens' queries, steep ones that raise their references often, leave a token's bits as they are."""
    import torch
    from webpytorch_amd import core
    q, cache, st = _case(71, T=T, NH=4, NKV=2, pos=500, lmax=2048)
    q = q.to(getattr(torch, dt))
    steep = q.clone()
    steep[::2] *= 40
    a, b = (core.attention_kv4(x, cache, st) for x in (q, steep))
    assert torch.equal(a[1::2], b[1::2]) and torch.isfinite(b).all()
    close(b, _torch_want(steep, cache, 500).cpu().numpy(), 1e-4 if dt == "float32" else 2 * F16_REL)


@pytest.mark.parametrize("size", [2e-6, 3e-5, 1e-3])
@pytest.mark.parametrize("T", [1, 700])
def test_values_below_the_normal_fp16_range(gpu, size, T):
    """Values that stand for fp16 subnormals, and keys of that size under a large scale, are not taken for zero."""
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(12)
    n, HD = 900, 64
    q = torch.randn((T, 2, HD), generator=g).cuda()
    k, v = (torch.randn((n, 1, HD), generator=g) * size for _ in range(2))
    cache = fill(k, v)
    got = core.attention_kv4(q, cache, state(torch, n - T), scale=0.125 / size)
    wk, wv = (t.cpu().numpy() for t in core.kv4_dequant(cache, 0, n))
    want = kv4.attention(q[-40:].cpu().numpy(), wk, wv, n - min(T, 40), float(np.float32(0.125 / size)))
    close(got[-40:], want, F32_REL)


@pytest.mark.parametrize("dt", ["float32", "float16"])
@pytest.mark.parametrize("T", [1, 3, 700])
def test_tensors_off_a_16_byte_line(gpu, T, dt):
    import torch
    from webpytorch_amd import core
    q, cache, st = _case(61, T=T, NH=2, NKV=1, pos=33, lmax=800)
    q = q.to(getattr(torch, dt))
    want = core.attention_kv4(q, cache, st)
    off = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)  # noqa: E731
    out = off(torch.zeros_like(q))
    core.attention_kv4(off(q), cache, st, out=out)
    assert torch.equal(out, want)
    cos, sin = tables(torch, 800, 64)
    qkv = torch.randn((T, 4 * 64), generator=torch.Generator().manual_seed(3)).to(q.dtype).cuda()
    a, b = core.kv4_cache(1, 800, 64), core.kv4_cache(1, 800, 64)
    assert torch.equal(core.qk_norm_rope(qkv, st, cos, sin, 2, a), core.qk_norm_rope(off(qkv), st, off(cos), off(sin), 2, b)) and torch.equal(a, b)
    with pytest.raises(ValueError, match="aligned"):
        core.attention_kv4(q, off(cache), st)


@pytest.mark.parametrize("T", [1, 5, 600])
def test_a_cache_that_ends_inside_a_block(gpu, T):
    """LMAX 45 through the C calls: positions from 45 on are not written, and tokens there attend up to 44."""
    import torch
    from webpytorch_amd import _lib, core
    g = torch.Generator().manual_seed(13)
    NH, NKV, HD, LMAX, pos = 4, 2, 64, 45, 30
    x = torch.randn((LMAX, (NH + 2 * NKV) * HD), generator=g).cuda()
    cos, sin = tables(torch, LMAX, HD)
    cache = core.kv4_cache(NKV, LMAX, HD)
    more = torch.randn((T + 20, (NH + 2 * NKV) * HD), generator=g).cuda()
    P, q0 = core.ptr, torch.empty((LMAX + T + 20, NH, HD), device="cuda")
    for rows, at in ((x, 0), (more, LMAX)):  # the second writes nothing
        _lib.call("miq_qk_norm_rope_kv4", P(rows), 0, rows.shape[1], None, None, 1e-6, P(state(torch, at)), P(cos), P(sin), P(q0), P(cache),
                  rows.shape[0], NH, NKV, HD, LMAX, None)
    assert not torch.stack(core.kv4_dequant(cache, LMAX, 64 - LMAX)).any()
    q, out = torch.randn((T, NH, HD), generator=g).cuda(), torch.empty((T, NH, HD), device="cuda")
    _lib.call("miq_attention_kv4", P(q), 0, P(cache), P(state(torch, pos)), P(out), T, NH, NKV, HD, LMAX, 0.125, None, 0, None)
    wk, wv = (t.cpu().numpy() for t in core.kv4_dequant(cache, 0, LMAX))
    close(out, kv4.attention(q.cpu().numpy(), wk, wv, pos, 0.125), F32_REL)


def test_argument_checks(gpu):
    import torch
    from webpytorch_amd import core
    q, cache, st = _case(41)
    with pytest.raises(ValueError, match="does not go with"):
        core.attention_kv4(q[:, :7], cache, st)
    with pytest.raises(TypeError, match="bfloat16"):
        core.attention_kv4(q.bfloat16(), cache, st)
    with pytest.raises(ValueError, match="contiguous"):
        core.attention_kv4(q, cache[:, ::2], st)
    with pytest.raises(ValueError, match="out is"):
        core.attention_kv4(q, cache, st, out=torch.empty((1, 8, 32), device="cuda"))
    with pytest.raises(ValueError, match="apart from q"):
        core.attention_kv4(q, cache, st, out=q)
    with pytest.raises(TypeError, match="state"):
        core.attention_kv4(q, cache, st.long())
    cos, sin = tables(torch, 4096, 64)
    qkv = torch.zeros((1, 12 * 64), device="cuda")
    with pytest.raises(ValueError, match="at least 4096"):
        core.qk_norm_rope(qkv, st, cos[:4000], sin, 8, cache)
    with pytest.raises(ValueError, match="query"):
        core.qk_norm_rope(qkv, st, cos, sin, 9, cache)
    with pytest.raises(ValueError, match="qn"):
        core.qk_norm_rope(qkv, st, cos, sin, 8, cache, qn=torch.ones(32, device="cuda"))
    with pytest.raises(TypeError, match="qkv"):
        core.qk_norm_rope(qkv.half(), st, cos, sin, 8, [torch.zeros((2, 4096, 64), device="cuda")] * 2)
    with pytest.raises(ValueError, match="positions"):
        core.kv4_dequant(cache, 4090, 7)
