"""GPU: reading back a whole 4-bit cache of more positions than a grid's second dimension has blocks for."""
import pytest

from test_gpu_kv4 import state

pytestmark = pytest.mark.gpu


def test_a_whole_long_cache(gpu):
    import torch
    from webpytorch_amd import core
    n, HD, T = 2_200_000, 64, 50
    cache = core.kv4_cache(1, n, HD)
    qkv = torch.randn((T, 3 * HD), generator=torch.Generator().manual_seed(1)).cuda()
    one, zero = torch.ones((cache.shape[1] * 32, HD // 2), device="cuda"), torch.zeros((cache.shape[1] * 32, HD // 2), device="cuda")
    for pos in (0, 1_000_003, n - T):
        core.qk_norm_rope(qkv, state(torch, pos), one, zero, 1, cache)
    k, v = core.kv4_dequant(cache)
    assert k.shape == v.shape == (1, cache.shape[1] * 32, HD)
    for pos in (0, 1_000_003, n - T):
        for whole, part in zip((k, v), core.kv4_dequant(cache, pos, T)):
            assert torch.equal(whole[:, pos:pos + T], part) and part.any()
    assert int((k != 0).any(-1).sum()) == int((v != 0).any(-1).sum()) == 3 * T
