"""GPU: QK-norm + RoPE + cache write where a wave takes several heads (from 8192 heads of all tokens on): head groups that
end inside q, between q and k, and between k and v."""
import numpy as np
import pytest

from oracle import kv4
from test_gpu_kv4 import state, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("NH,NKV,HD", [(14, 2, 64), (3, 1, 80), (9, 3, 128), (7, 7, 192), (6, 2, 256), (5, 5, 2)])
@pytest.mark.parametrize("norm", ["qk", "q", "k", ""])
@pytest.mark.parametrize("more", [0, 1, 300])
def test_fp32_cache_is_the_two_calls_bit_for_bit(gpu, NH, NKV, HD, norm, more):
    import torch
    from webpytorch_amd import _lib, core
    g = torch.Generator().manual_seed(more + HD)
    heads, pos = NH + 2 * NKV, 5
    T = 8191 // heads + more  # the last count below the border, the first from it on, and further
    W, LMAX = heads * HD, pos + T - 2
    qkv = torch.randn((T, W + 3), generator=g).cuda()[:, :W]
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
@pytest.mark.parametrize("NH,NKV,HD", [(15, 3, 64), (7, 1, 128), (5, 5, 192), (9, 3, 256)])
@pytest.mark.parametrize("norm,more", [("qk", 0), ("qk", 1), ("", 40), ("k", 40)])
def test_kv4_write_matches_float64(gpu, NH, NKV, HD, norm, more, dt):
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(more + HD)
    T, pos = 8191 // (NH + NKV) + more, 45
    lmax = (pos + T + 31) // 32 * 32
    qkv = (torch.randn((T, (NH + 2 * NKV) * HD), generator=g) * 2).to(getattr(torch, dt))
    qn, kn = (1 + 0.3 * torch.randn(HD, generator=g) if c in norm else None for c in "qk")
    before = torch.randint(0, 256, (NKV, lmax // 32, 40 * HD), dtype=torch.uint8, generator=g)
    cache = before.cuda()
    cos, sin = tables(torch, lmax, HD)
    q = core.qk_norm_rope(qkv.cuda(), state(torch, pos), cos, sin, NH, cache, qn=None if qn is None else qn.cuda(),
                          kn=None if kn is None else kn.cuda())
    x = qkv.float().numpy().reshape(T, -1, HD)
    c, s = (t[pos:pos + T].cpu().numpy() for t in (cos, sin))
    wq = kv4.norm_rope(x[:, :NH], None if qn is None else qn.numpy(), c, s)
    wk = kv4.norm_rope(x[:, NH:NH + NKV], None if kn is None else kn.numpy(), c, s).astype(np.float32)
    ulp = 2.0 ** (-24 if dt == "float32" else -11)  # half a step, and fp16's smallest half step below its normal range
    assert (np.abs(q.double().cpu().numpy() - wq) <= ulp * np.abs(wq) * 1.001 + 2.0 ** -25).all()
    was, now = kv4.unpack(before.numpy(), lmax), kv4.unpack(cache.cpu().numpy(), lmax)
    at = np.arange(pos, pos + T)
    rest = np.setdiff1d(np.arange(lmax), at)
    for part, rows in ((0, wk), (1, x[:, NH + NKV:])):
        want = kv4.quantize(np.ascontiguousarray(rows.transpose(1, 0, 2)))
        for i in range(3):
            assert np.array_equal(now[part][i][:, at], want[i], equal_nan=i > 0)
            view = (lambda t: t) if i == 0 else (lambda t: np.ascontiguousarray(t).view(np.uint16))
            assert np.array_equal(view(now[part][i])[:, rest], view(was[part][i])[:, rest])


@pytest.mark.parametrize("HD,T", [(64, 2000), (128, 1000), (192, 30), (256, 700)])
def test_fp16_queries_are_rounded_once(gpu, HD, T):
    """Without a norm a query is two fp64 products and their sum: the fp16 number next to it, not that of its fp32
    number (a value in 2^13 or so lies between the two roundings)."""
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(HD)
    NH, lmax = 8, (T + 31) // 32 * 32
    qkv = torch.randn((T, (NH + 2) * HD), generator=g).half()
    cache = core.kv4_cache(1, lmax, HD)
    cos, sin = tables(torch, lmax, HD)
    q = core.qk_norm_rope(qkv.cuda(), state(torch, 0), cos, sin, NH, cache)
    x = qkv.numpy().reshape(T, -1, HD)[:, :NH].astype(np.longdouble)
    c, s = (t[:T].cpu().numpy().astype(np.longdouble)[:, None] for t in (cos, sin))
    h = HD // 2  # 11 x 24 bits a product: 64 bits hold the sum but for cancellation's last ones
    want = np.concatenate([x[..., :h] * c - x[..., h:] * s, x[..., h:] * c + x[..., :h] * s], -1)
    lo, hi = (np.nextafter(want.astype(np.float16), np.float16(d)).astype(np.longdouble) for d in (-np.inf, np.inf))
    got = q.cpu().numpy().astype(np.longdouble)
    # the nearest: no neighbour is nearer by more than fp64's own rounding of the sum
    err, slack = np.abs(got - want), np.abs(want) * 2.0 ** -50 + 2.0 ** -60
    assert (err <= np.minimum(np.abs(lo - want), np.abs(hi - want)) + slack).all()
