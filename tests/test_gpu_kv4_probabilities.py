"""GPU: the bits that the probabilities of attention over the 4-bit cache carry."""
import math

import pytest

from test_gpu_kv4 import fill, state

pytestmark = pytest.mark.gpu


def last_rows(q, cache, pos, rows):
    """float64 of the last `rows` tokens."""
    import torch
    from webpytorch_amd import core
    T, NH, HD = q.shape
    n = pos + T
    k, v = (t.double() for t in core.kv4_dequant(cache, 0, n))
    out = torch.empty((rows, NH, HD), dtype=torch.float64, device="cuda")
    later = torch.arange(n, device="cuda")[None, :] > n - rows + torch.arange(rows, device="cuda")[:, None]
    for h in range(NH):
        s = torch.mm(q[-rows:, h].double(), k[h // (NH // k.shape[0])].t().contiguous()) / math.sqrt(HD)
        s[later] = -math.inf
        out[:, h] = torch.mm(torch.softmax(s, 1), v[h // (NH // k.shape[0])])
    return out


@pytest.mark.parametrize("NH,NKV,HD", [(4, 2, 64), (4, 1, 128), (2, 1, 192), (2, 1, 256)])
@pytest.mark.parametrize("T,pos,lmax", [(1, 700, 701), (20, 5000, 8192), (700, 0, 700), (90, 4000, 70000)])
def test_fp16_rows_are_off_by_their_own_rounding(gpu, NH, NKV, HD, T, pos, lmax):
    """fp16 queries are exact operands and probabilities have 22 bits, so that an output is the fp16 number
    next to the exact one: half a step of it, and 1e-5 of the row's size for the 22 bits and fp32 sums."""
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(T + HD)
    q = torch.randn((T, NH, HD), generator=g).half().cuda()
    k, v = (torch.randn((pos + T, NKV, HD), generator=g) for _ in range(2))
    cache = fill(k, v, lmax=lmax)
    rows = min(T, 64)
    got = core.attention_kv4(q, cache, state(torch, pos))[-rows:].double()
    want = last_rows(q, cache, pos, rows)
    size = want.pow(2).mean(-1, keepdim=True).sqrt()
    assert float(((got - want).abs() - 2.0 ** -11 * want.abs() - 2.0 ** -25 - 1e-5 * size).max()) <= 0
