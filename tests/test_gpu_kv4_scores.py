"""GPU: attention over the 4-bit cache where scores are far from 1: steep queries, scores past any integer that fp32
holds, rows that pass from moderate to far scores, and rows without a finite score."""
import math

import numpy as np
import pytest

from test_gpu_kv4 import fill, state

pytestmark = pytest.mark.gpu

# of a row whose probability is one key's (the others' below e^-20 together): the key's p as two fp16 numbers and its sum
# of the same two, each product rounded to fp32 once, and the quotient
ONE_KEY = 4 * 2.0 ** -24


def check(got, q, cache, pos, scale, f32):
    """Rows that one key decides (its score is ahead of the others' by more than what q's 22 bits and fp32 sums
    leave open, and by 20 + ln of their number) hold that key's value; the others lie within their values' range. Returns
    the decided rows' share."""
    import torch
    from webpytorch_amd import core
    T, NH, HD = q.shape
    n = max(pos + T, 1)
    k, v = (t.double() for t in core.kv4_dequant(cache, 0, n))
    rep = NH // k.shape[0]
    assert torch.isfinite(got).all()
    decided = 0
    for h in range(NH):
        kk, vv, qq = k[h // rep], v[h // rep], q[:, h].double()
        s = torch.mm(qq, kk.t().contiguous()) * scale
        size = torch.mm((qq.abs().amax(1, keepdim=True).expand_as(qq) if f32 else qq.abs()).contiguous(), kk.abs().t().contiguous()) * abs(scale)
        open_ = size.amax(1) * 2.0 ** -20  # q's 2^-22 of the row's largest value, HD / 32 sums of fp32
        s[torch.arange(n, device="cuda")[None, :] > pos + torch.arange(T, device="cuda")[:, None]] = -math.inf
        top = torch.topk(s, min(2, n), 1)
        ahead = top.values[:, 0] - (top.values[:, 1] if n > 1 else -math.inf)
        sure = ahead > 2 * open_ + 20 + math.log(n)
        decided += int(sure.sum())
        want = vv[top.indices[:, 0]]
        g = got[:, h].double()
        tol = (ONE_KEY + (0 if f32 else 2.0 ** -11)) * vv.abs().max() + math.exp(-20) * vv.abs().max()
        assert float((g - want).abs()[sure].max()) <= tol, (h, float((g - want).abs()[sure].max()))
        assert float(g.max()) <= float(vv.max()) + tol and float(g.min()) >= float(vv.min()) - tol
    return decided / (T * NH)


@pytest.mark.parametrize("NH,NKV,HD", [(4, 2, 64), (4, 1, 128), (2, 1, 256)])
@pytest.mark.parametrize("T,pos,lmax", [(1, 0, 64), (3, 900, 4096), (1, 20000, 20001), (300, 0, 300), (300, 700, 8192), (80, 30000, 70000)])
@pytest.mark.parametrize("size", [1e5, 3e8, 1e10, 1e12, 1e30])
def test_large_queries(gpu, NH, NKV, HD, T, pos, lmax, size):
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(T + HD)
    n = pos + T
    q = (torch.randn((T, NH, HD), generator=g) * size).cuda()
    k, v = (torch.randn((n, NKV, HD), generator=g) for _ in range(2))
    cache = fill(k, v, lmax=lmax)
    share = check(core.attention_kv4(q, cache, state(torch, pos)), q, cache, pos, 1 / math.sqrt(HD), True)
    assert share > 0.8


@pytest.mark.parametrize("T,pos", [(1, 0), (3, 900), (300, 0), (300, 700)])
@pytest.mark.parametrize("HD", [64, 128])
def test_large_fp16_queries_and_saturated_keys(gpu, HD, T, pos):
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(T + HD)
    q = (torch.randn((T, 4, HD), generator=g) * 2e4).clamp(-6e4, 6e4).half().cuda()
    k, v = torch.randn((pos + T, 2, HD), generator=g) * 9000, torch.randn((pos + T, 2, HD), generator=g)
    cache = fill(k, v, lmax=4096)
    share = check(core.attention_kv4(q, cache, state(torch, pos)), q, cache, pos, 1 / math.sqrt(HD), False)
    assert share > 0.8


@pytest.mark.parametrize("T,pos,lmax", [(1, 1500, 2000), (700, 800, 1500), (90, 9000, 40000)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("size", [1e6, 1e9, 1e11])
def test_scores_that_grow_along_the_cache(gpu, T, pos, lmax, sign, size):
    """From moderate to far (positive) and from far to moderate (negative): each position's score is the highest
    yet, so that the reference moves in every block."""
    import torch
    from webpytorch_amd import core
    HD, n = 64, pos + T
    g = torch.Generator().manual_seed(7)
    k = torch.zeros((n, 1, HD))
    ramp = torch.linspace(0, 1, n) ** 3
    k[:, 0, :32] = (ramp if sign > 0 else ramp - 1)[:, None]  # one value a group: exact but for S and Z's roundings
    v = torch.randn((n, 1, HD), generator=g)
    q = torch.zeros((T, 2, HD))
    q[:, :, 0] = size
    q = q.cuda()
    cache = fill(k, v, lmax=lmax)
    check(core.attention_kv4(q, cache, state(torch, pos)), q, cache, pos, 1 / 8, True)


@pytest.mark.parametrize("dt", ["float32", "float16"])
@pytest.mark.parametrize("T,lmax", [(5, 2048), (40, 2048), (700, 2048), (90, 70000)])
def test_moderate_rows_beside_far_ones(gpu, T, lmax, dt):
    """Neighbours with far scores leave a token's bits as they are."""
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(T)
    HD, pos, big = 64, 500, 1e10 if dt == "float32" else 3e4
    q = torch.randn((T, 4, HD), generator=g)
    k, v = torch.randn((pos + T, 2, HD), generator=g) * (1 if dt == "float32" else 1000), torch.randn((pos + T, 2, HD), generator=g)
    cache = fill(k, v, lmax=lmax)
    far = q.clone()
    far[::2] = (far[::2] * big).clamp(-1e30 if dt == "float32" else -6e4, 1e30 if dt == "float32" else 6e4)
    a, b = (core.attention_kv4(x.to(getattr(torch, dt)).cuda(), cache, state(torch, pos)) for x in (q, far))
    assert torch.equal(a[1::2], b[1::2]) and torch.isfinite(b).all() and b.abs().amax(-1).min() > 0


@pytest.mark.parametrize("T,pos,lmax", [(1, 40, 64), (1, 5000, 5001), (40, 0, 64), (700, 0, 700), (90, 3000, 70000)])
def test_rows_whose_scores_are_all_minus_infinity(gpu, T, pos, lmax):
    """An infinity in a query times keys of one sign: the softmax of -inf alone is not a number, and zeros are for
    rows without a key."""
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(3)
    HD, n = 64, pos + T
    k, v = torch.randn((n, 1, HD), generator=g), torch.randn((n, 1, HD), generator=g)
    k[..., 5] = -4 - torch.rand((n, 1), generator=g)
    q = torch.randn((T, 2, HD), generator=g).half()
    q[::3, 0, 5] = math.inf
    got = core.attention_kv4(q.cuda(), fill(k, v, lmax=lmax), state(torch, pos))
    assert torch.isnan(got[::3, 0]).all() and torch.isfinite(got[:, 1]).all()
    rest = torch.arange(T) % 3 != 0
    assert torch.isfinite(got[rest]).all()


@pytest.mark.parametrize("size,scale", [(3e-39, 3e37), (2e-42, 2e37), (1e-37, 1e36)])
@pytest.mark.parametrize("T", [1, 700])
def test_queries_below_the_normal_fp32_range(gpu, T, size, scale):
    """Under a scale that makes scores of them (the second pair: queries of some thousand steps of 2^-149)."""
    import torch
    from test_gpu_kv4_probabilities import last_rows
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(T)
    HD, pos = 64, 600
    q = (torch.randn((T, 2, HD), generator=g) * size).cuda()
    k, v = (torch.randn((pos + T, 1, HD), generator=g) for _ in range(2))
    cache = fill(k, v)
    rows = min(T, 32)
    got = core.attention_kv4(q, cache, state(torch, pos), scale=scale)[-rows:].double()
    want = last_rows(q.double() * (scale * math.sqrt(HD)), cache, pos, rows)  # which divides by sqrt(HD)
    assert float((got - want).norm() / want.norm()) <= 5e-6
