"""GPU: the probabilities of attention over the 4-bit cache. Small ones count too: a first key that takes most of the
softmax and has a small value (an attention sink) leaves the output to many small probabilities."""
import math

import pytest

from test_gpu_kv4 import fill, state

pytestmark = pytest.mark.gpu

# A probability is held as two fp16 numbers of 2^11 p, to 2^-25 at the least: of 16000 keys that share 1 % it is 2^11 x 6e-7
# = 2^-9.6, so 2^-15 of each, at random, 2^-22 of their sum. The scores are exact where they are large (the sink's), and
# fp32 sums of 500 steps stay within 500 x 2^-24 / 6.
SINK_REL = 5e-6


def sink(n, nkv, HD, share, g):
    """Keys and values (n, nkv, HD): position 0 takes `share` of every query that `queries` makes."""
    import torch
    k, v = torch.randn((n, nkv, HD), generator=g), 1 + torch.randn((n, nkv, HD), generator=g)
    k[:, :, :32] = 0
    # e^score of the others sums to n e^(1/2 (HD - 32) / HD): the queries' scores are N(0, (HD - 32) / HD)
    k[0] = 0
    k[0, :, :32] = (math.log(n) + 0.5 * (HD - 32) / HD + math.log(share / (1 - share))) * math.sqrt(HD) / 32
    v[0] *= 0.01
    return k, v


def queries(T, NH, HD, g):
    import torch
    q = torch.randn((T, NH, HD), generator=g)
    q[:, :, :32] = 1
    return q


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


@pytest.mark.parametrize("share", [0.9, 0.99, 0.999])
@pytest.mark.parametrize("T,n,NH,NKV,HD", [(1, 16000, 4, 2, 64), (30, 16000, 2, 1, 64), (4096, 6000, 8, 8, 64), (4096, 16000, 8, 8, 64),
                                           (2048, 16000, 16, 16, 128), (100, 100000, 4, 4, 64)])
def test_sink_keys(gpu, T, n, NH, NKV, HD, share):
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(n)
    k, v = sink(n, NKV, HD, share, g)
    q = queries(T, NH, HD, g).cuda()
    cache = fill(k, v)
    rows = min(T, 16)
    got = core.attention_kv4(q, cache, state(torch, n - T))[-rows:].double()
    want = last_rows(q, cache, n - T, rows)
    err = float((got - want).norm() / want.norm())
    assert err <= SINK_REL, err


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
