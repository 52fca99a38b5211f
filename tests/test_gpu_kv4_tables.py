"""GPU: rotation tables of a context that ends inside a block of the 4-bit cache."""
import pytest

from test_gpu_kv4 import state, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lmax", [1, 33, 45, 64])
@pytest.mark.parametrize("short", ["cos", "sin", "both"])
def test_tables_as_long_as_the_context(gpu, lmax, short):
    import torch
    from webpytorch_amd import core
    NH, NKV, HD, T = 4, 2, 64, 70
    qkv = torch.randn((T, (NH + 2 * NKV) * HD), generator=torch.Generator().manual_seed(lmax)).cuda()
    a, b = core.kv4_cache(NKV, lmax, HD), core.kv4_cache(NKV, lmax, HD)
    cos, sin = tables(torch, a.shape[1] * 32, HD)
    cut = [t[:lmax].contiguous() if short in (n, "both") else t for n, t in (("cos", cos), ("sin", sin))]
    got = core.qk_norm_rope(qkv, state(torch, 0), *cut, NH, a)
    want = core.qk_norm_rope(qkv[:lmax], state(torch, 0), cos, sin, NH, b)
    n = min(T, lmax)
    assert torch.equal(got[:n], want[:n]) and not got[n:].any() and torch.equal(a, b)
    if lmax > 32:
        with pytest.raises(ValueError, match="at least 64"):
            core.qk_norm_rope(qkv, state(torch, 0), cos[:32].contiguous(), sin, NH, a)
