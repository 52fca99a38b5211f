"""GPU: outputs that share memory with what other workgroups still read are refused, wherever they start, and views that
only share a storage are not."""
import pytest

from test_gpu_kv4 import fill, state, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["float32", "float16"])
def test_attention(gpu, dt):
    import torch
    from webpytorch_amd import core
    T, NH, HD = 3, 4, 64
    n = T * NH * HD
    pool = torch.randn(3 * n, generator=torch.Generator().manual_seed(1)).to(getattr(torch, dt)).cuda()
    cache = fill(*(torch.randn((40, 2, HD)) for _ in range(2)))
    at = lambda a: pool[a:a + n].view(T, NH, HD)  # noqa: E731
    q, st = at(n), state(torch, 30)
    want = core.attention_kv4(q, cache, st)
    for a in (1, n - HD, n, n + 1, n + HD, 2 * n - 1):
        with pytest.raises(ValueError, match="apart from q"):
            core.attention_kv4(q, cache, st, out=at(a))
    for a in (0, 2 * n):
        assert torch.equal(core.attention_kv4(q, cache, st, out=at(a)), want)
    inside = cache.view(-1).view(q.dtype)
    with pytest.raises(ValueError, match="apart from"):
        core.attention_kv4(q, cache, st, out=inside[8:8 + n].view(T, NH, HD))


@pytest.mark.parametrize("four", [True, False])
@pytest.mark.parametrize("T", [1, 3])
def test_norm_rope(gpu, four, T):
    import torch
    from webpytorch_amd import core
    NH, NKV, HD, lmax, gap = 4, 2, 64, 64, 512
    W, n = (NH + 2 * NKV) * HD, T * NH * HD
    pool = torch.randn(4 * (T * (W + gap) + n), generator=torch.Generator().manual_seed(2)).cuda()
    cos, sin = tables(torch, lmax, HD)
    st, start = state(torch, 5), 2 * n
    qkv = pool[start:start + T * (W + gap)].view(T, W + gap)[:, :W]
    new = lambda: core.kv4_cache(NKV, lmax, HD) if four else [torch.zeros((NKV, lmax, HD), device="cuda") for _ in range(2)]  # noqa: E731
    want = core.qk_norm_rope(qkv, st, cos, sin, NH, new())
    at = lambda a: pool[a:a + n].view(T, NH, HD)  # noqa: E731
    end = start + (T - 1) * (W + gap) + W
    for a in (start - n + 1, start - 1, start, start + HD, end - 1):
        with pytest.raises(ValueError, match="apart from qkv"):
            core.qk_norm_rope(qkv, st, cos, sin, NH, new(), out=at(a))
    for a in (start - n, end):
        assert torch.equal(core.qk_norm_rope(qkv, st, cos, sin, NH, new(), out=at(a)), want)
    if T == 1:  # between two rows of a wider tensor
        return
    two = pool[start:start + 2 * (W + 2 * n)].view(2, W + 2 * n)[:, :W]
    want = core.qk_norm_rope(two, st, cos, sin, NH, new())
    out = pool[start + W:start + W + 2 * NH * HD].view(2, NH, HD)
    assert torch.equal(core.qk_norm_rope(two, st, cos, sin, NH, new(), out=out), want)


def test_caches(gpu):
    """The two fp32 caches, and either of them with the rows or the output."""
    import torch
    from webpytorch_amd import core
    NH, NKV, HD, lmax = 4, 2, 64, 64
    cos, sin = tables(torch, lmax, HD)
    n, W = NKV * lmax * HD, (NH + 2 * NKV) * HD
    pool = torch.zeros(3 * n, device="cuda")
    kc = pool[n:2 * n].view(NKV, lmax, HD)
    st, qkv = state(torch, 0), torch.zeros((1, W), device="cuda")
    for vc in (kc, pool[n - HD:2 * n - HD].view(NKV, lmax, HD), pool[2 * n - 1:3 * n - 1].view(NKV, lmax, HD)):
        for pair in ((kc, vc), (vc, kc)):
            with pytest.raises(ValueError, match="caches overlap"):
                core.qk_norm_rope(qkv, st, cos, sin, NH, pair)
    vc = pool[2 * n:].view(NKV, lmax, HD)
    core.qk_norm_rope(qkv, st, cos, sin, NH, (kc, vc))
    with pytest.raises(ValueError, match="apart from"):
        core.qk_norm_rope(qkv, st, cos, sin, NH, (kc, vc), out=vc.view(-1)[64:64 + NH * HD].view(1, NH, HD))
    with pytest.raises(ValueError, match="apart from"):
        core.qk_norm_rope(kc.view(-1)[:W].view(1, W), st, cos, sin, NH, (kc, vc))
    four = core.kv4_cache(NKV, lmax, HD)
    inside = four.view(-1).view(torch.float32)
    with pytest.raises(ValueError, match="apart from"):
        core.qk_norm_rope(qkv, st, cos, sin, NH, four, out=inside[4:4 + NH * HD].view(1, NH, HD))
    with pytest.raises(ValueError, match="apart from"):
        core.qk_norm_rope(inside[:W].view(1, W), st, cos, sin, NH, four)
