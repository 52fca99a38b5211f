"""GPU: the serving operators on two streams at a time, each stream's results counted by itself: a wrong one cannot be lost to the other stream's
store."""
import pytest

pytestmark = pytest.mark.gpu


def test_two_streams_count_their_own(gpu):
    """Attention in parts (workspaces of the streams) and verification (two launches through one), against the same calls alone."""
    import torch
    from webpytorch_amd import core
    sets = []
    for i in range(2):
        g = torch.Generator(device="cuda").manual_seed(i)
        n, P = 6000 + 1000 * i, 32
        pages = torch.randperm(300, device="cuda", generator=g)[:(n + P - 1) // P].to(torch.int32)[None].contiguous()
        cache = torch.randn((300, 2, 2, P, 64), device="cuda", generator=g).half()
        q = torch.randn((1, 2, 4, 64), device="cuda", generator=g)
        pos = torch.tensor([[n - 2, n - 1]], dtype=torch.int32, device="cuda")
        x, d = (torch.randn((3, r, 20000 + i), device="cuda", generator=g) * 3 for r in (3, 2))
        ids = d.argmax(-1).to(torch.int32)
        u = torch.rand((3, 3), device="cuda", generator=g)
        sets.append(((q, pos, pages, cache), (x, ids, u, d)))
    calls = [lambda s=s: (core.paged_attention(*s[0]), *core.verify_drafts(*s[1])) for s in sets]
    alone = [c() for c in calls]
    streams = [torch.cuda.Stream() for _ in sets]
    wrong = [torch.zeros((), dtype=torch.int64, device="cuda") for _ in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, c, want, w in zip(streams, calls, alone, wrong):
            with torch.cuda.stream(st):
                for a, b in zip(c(), want):
                    w += (a != b).sum()
    torch.cuda.synchronize()
    assert [int(w) for w in wrong] == [0, 0]
