"""GPU: log probabilities of given tokens, entropy, ranks and alternatives against float64."""
import math

import numpy as np
import pytest

from oracle import kv4

pytestmark = pytest.mark.gpu


def check(x, ids, k, got=None):
    """Floats: lse is 2^-24 of itself plus the error of an fp32 sum over a thread's values (under 2^-20
    relatively); entropy likewise, its two terms up to log V; whole numbers equal."""
    import torch
    from webpytorch_amd import core
    got = got or core.token_logprobs(x, ids, k)
    want = kv4.token_logprobs(x.float().cpu().numpy(), ids.cpu().numpy(), k)
    size = 1 + math.log(x.shape[1])
    for g, w in zip(got, want):
        g = g.cpu().numpy()
        assert g.shape == w.shape
        if g.dtype == np.int32:
            assert np.array_equal(g, w)
            continue
        fine = np.isfinite(w)
        assert np.array_equal(np.isnan(g), np.isnan(w)) and np.array_equal(g[~fine & ~np.isnan(w)], w[~fine & ~np.isnan(w)])
        assert (np.abs(g[fine] - w[fine]) <= 2.0 ** -20 * size + 2.0 ** -23 * np.abs(w[fine])).all()
    return got


@pytest.mark.parametrize("dt", ["float32", "float16"])
@pytest.mark.parametrize("T,V,pad,k", [(1, 1, 0, 1), (1, 151936, 0, 5), (3, 7, 2, 7), (2, 4096, 0, 32), (5, 4097, 3, 20), (9, 32003, 61, 8),
                                       (40, 1000, 1, 0), (1030, 515, 0, 3), (2, 65537, 5, 32), (17, 33, 0, 32)])
def test_matches_float64(gpu, T, V, pad, k, dt):
    import torch
    g = torch.Generator().manual_seed(V + T)
    x = (torch.randn((T, V + pad), generator=g) * 3).to(getattr(torch, dt)).cuda()[:, :V]
    ids = torch.randint(0, V, (T,), generator=g, dtype=torch.int32).cuda()
    check(x, ids, k)
    if pad:  # rows that start off a 16-byte line
        y = torch.empty(x.numel() + 3, dtype=x.dtype, device="cuda")[3:].view(T, V).copy_(x)
        check(y, ids.long(), k)


@pytest.mark.parametrize("make", ["equal", "up", "down", "two", "zeros"])
def test_ties_and_sorted_rows(gpu, make):
    """Equal logits go by their index, -0 is 0; rows sorted up or down fill the candidates' buffer."""
    import torch
    V = 30011
    r = {"equal": torch.full((V,), 1.5), "up": torch.arange(V) * 1e-3, "down": torch.arange(V) * -1e-3,
         "two": (torch.arange(V) % 7 == 3).float() * 2, "zeros": torch.where(torch.arange(V) % 2 == 0, -0.0, 0.0)}[make]
    for T in (2, 1100):
        x = r.float().repeat(T, 1)[:, :V if T == 2 else 4200].contiguous().cuda()
        ids = torch.full((T,), 77, dtype=torch.int32, device="cuda")
        check(x[:2], ids[:2], 32)
        if T > 2:
            from webpytorch_amd import core
            got = core.token_logprobs(x, ids, 32)
            for a, b in zip(got, core.token_logprobs(x[:1], ids[:1], 32)):
                # other segments, so other sums
                assert torch.allclose(a[0], b[0], rtol=1e-6) and all(torch.equal(a[i], a[0]) for i in (1, 600, T - 1))


def test_masked_and_non_finite_rows(gpu):
    import torch
    inf, nan, V = math.inf, math.nan, 9001
    x = torch.randn((9, V), generator=torch.Generator().manual_seed(4))
    x[0, 1:] = -inf                          # one token left
    x[1] = -inf                              # none
    x[2, ::2] = -inf
    x[3, 100] = nan
    x[4, 100] = inf
    x[5] = nan
    x[6, :] = torch.finfo(torch.float32).min  # masked by the type's lowest value, all of it
    x[7, 5:] = torch.finfo(torch.float32).min
    x[8] *= 1e4
    ids = torch.tensor([0, 3, 0, 100, 100, 2, 8, 4, 1], dtype=torch.int32, device="cuda")
    got = check(x.cuda(), ids, 6)
    assert list(got.top_ids[1].cpu()) == [0, 1, 2, 3, 4, 5] and float(got.entropy[1]) == 0.0
    check(x.cuda(), ids.roll(1), 20)


def test_ids_outside_the_vocabulary(gpu):
    import torch
    x = torch.randn((5, 300), generator=torch.Generator().manual_seed(4)).cuda()
    got = check(x, torch.tensor([-1, 300, -100, 2 ** 31 - 1, 5], dtype=torch.int32, device="cuda"), 2)
    assert got.logprobs[:4].tolist() == [0.0] * 4 and got.ranks[:4].tolist() == [-1] * 4
    big = torch.tensor([2 ** 32 + 5, -2 ** 40, 1, 2, 3], device="cuda")
    from webpytorch_amd import core
    got = core.token_logprobs(x, big)
    assert got.ranks[:2].tolist() == [-1, -1] and got.top_ids.shape == (5, 0)


def test_deterministic_in_graphs_and_on_streams(gpu):
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(8)
    cases = [(torch.randn((T, 50000), generator=g).cuda(), torch.randint(0, 50000, (T,), generator=g, dtype=torch.int32).cuda())
             for T in (1, 6)]
    want = [core.token_logprobs(*c, 20) for c in cases]
    graphs, outs = [], []
    for c in cases:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(core.token_logprobs(*c, 20))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for _ in range(4):
            for gr, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    gr.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, w))
        assert all(torch.equal(a, b) for a, b in zip(core.token_logprobs(*cases[1], 20), want[1]))


def test_more_rows_than_one_launch_takes(gpu):
    import torch
    g = torch.Generator().manual_seed(9)
    x, ids = torch.randn((70001, 9), generator=g).cuda(), torch.randint(0, 9, (70001,), generator=g, dtype=torch.int32).cuda()
    from webpytorch_amd import core
    got = core.token_logprobs(x, ids, 3)
    want = torch.log_softmax(x.double(), 1)
    assert float((got.logprobs - want.gather(1, ids.long()[:, None])[:, 0]).abs().max()) < 1e-5
    assert torch.equal(got.top_ids, torch.sort(x, dim=1, descending=True, stable=True).indices[:, :3].int())


def test_row_of_the_decode_state(gpu):
    import torch
    from webpytorch_amd import _lib, core
    V, k, rows = 20000, 4, 6
    x = torch.randn((1, V), generator=torch.Generator().manual_seed(8)).cuda()
    ids = torch.tensor([77], dtype=torch.int32, device="cuda")
    want = core.token_logprobs(x, ids, k)
    ws = torch.zeros(core.token_logprobs_workspace_bytes(1, V, k), dtype=torch.uint8, device="cuda")
    outs = [torch.full((rows,) + t.shape[1:], 9, dtype=t.dtype, device="cuda") for t in want]
    for step in (4, 0, 7, 6):
        st = torch.tensor([0, step, 0, 0], dtype=torch.int32, device="cuda")
        _lib.call("miq_token_logprobs", core.ptr(x), 0, V, core.ptr(ids), 1, V, k, *(core.ptr(o) for o in outs), core.ptr(st), rows,
                  core.ptr(ws), ws.numel(), core.stream_handle())
    for o, w in zip(outs, want):
        assert torch.equal(o[3], w[0]) and torch.equal(o[5], w[0])
        assert all((o[r] == 9).all() for r in (0, 1, 2, 4))


def test_argument_checks(gpu):
    import torch
    from webpytorch_amd import core
    x, ids = torch.zeros((3, 40), device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    for bad, exc in (((x, ids[:2]), ValueError), ((x, ids, 33), ValueError), ((x[:, :4], ids, 5), ValueError), ((x.double(), ids), TypeError),
                     ((x[0], ids), ValueError), ((x, ids.float()), TypeError), ((x, ids.cpu()), ValueError)):
        with pytest.raises(exc):
            core.token_logprobs(*bad)
    assert core.token_logprobs(x[:0], ids[:0], 3).top_ids.shape == (0, 3)
    t = torch.randn((40, 3), device="cuda").t()  # columns apart
    check(t, ids, 5)
