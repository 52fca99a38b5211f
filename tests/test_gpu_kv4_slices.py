"""GPU: attention of few rows over a 4-bit cache of several slices, with random keys, against float64: every head
dimension and type of rows, several blocks a wave, and a cache whose length leaves more slices than its positions use."""
import pytest

from test_gpu_kv4 import F16_REL, F32_REL, close, fill, state
from test_gpu_kv4_probabilities import last_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["float32", "float16"])
@pytest.mark.parametrize("NH,NKV,HD", [(6, 2, 64), (4, 1, 128), (3, 1, 192), (4, 2, 256)])
@pytest.mark.parametrize("T,pos,lmax", [(1, 900, 1000), (5, 900, 40000), (16, 5000, 5016), (1, 5000, 70000), (5, 20000, 20005), (16, 20000, 130000),
                                        (1, 20001, 33000)])
def test_few_rows_in_slices(gpu, NH, NKV, HD, T, pos, lmax, dt):
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(pos + T + HD)
    n = pos + T
    q = torch.randn((T, NH, HD), generator=g).to(getattr(torch, dt)).cuda()
    k, v = (torch.randn((n, NKV, HD), generator=g) for _ in range(2))
    k[torch.randint(0, n, (60,), generator=g)] *= 3  # some keys stand out, wherever they are
    rnd = torch.randint(0, 256, (NKV, (lmax + 31) // 32, 40 * HD), dtype=torch.uint8, generator=g).cuda()
    cache = fill(k, v, cache=rnd)
    got = core.attention_kv4(q, cache, state(torch, pos))
    close(got, last_rows(q, cache, pos, T).cpu().numpy(), F32_REL if dt == "float32" else F16_REL)
