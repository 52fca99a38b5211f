"""GPU: attention over a paged cache against float64 (`oracle/paged.py`): types, head layouts, lengths, pages, masks,
non-finite values, splits, graphs, streams and far offsets."""
import threading

import numpy as np
import pytest

from oracle import paged

pytestmark = pytest.mark.gpu

# q (fp32 rows) and p as two fp16 numbers keep 2^-22 of each, fp32 sums of the products the rest: of the output's norm
F32_REL = 5e-6
F16_REL = 2.0 ** -11  # half a step of fp16


def setup(torch, seed, lens, T, NH, NKV, HD, P, x, cache, extra=2):
    """q, positions (the last T of lens[s] each; -1 ahead of 0), a page table in random order, the cache (NaN in unused pages)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // P) for n in lens]
    num, most = sum(need) + extra, max(1, max(need))
    order = torch.randperm(num, generator=g).to(torch.int32)
    pages, at = torch.full((len(lens), most), -1, dtype=torch.int32), 0
    c = torch.randn((num, 2, NKV, P, HD), generator=g).to(getattr(torch, cache))
    for s, n in enumerate(need):
        pages[s, :n] = order[at:at + n]
        at += n
        if lens[s] % P:
            c[pages[s, n - 1].item(), :, :, lens[s] % P:] = float("nan")
    for p in order[at:].tolist():
        c[p] = float("nan")
    q = torch.randn((len(lens), T, NH, HD), generator=g).to(getattr(torch, x))
    pos = (torch.tensor(lens, dtype=torch.int32)[:, None] - T + torch.arange(T, dtype=torch.int32)[None]).clamp(min=-1)
    return q, pos, pages, c


def check(got, q, pos, pages, c, scale=None, rel=F32_REL):
    want, mag, _ = paged.attention(q.numpy(), pos.numpy(), pages.numpy(), c.numpy(), scale)
    got = got.double().cpu().numpy()
    assert got.shape == want.shape and np.isfinite(got).all()
    half = q.numpy().dtype == np.float16
    err = np.abs(got - want)
    assert np.linalg.norm(err) <= (rel + (F16_REL if half else 0)) * np.linalg.norm(want) + 1e-30, np.linalg.norm(err) / np.linalg.norm(want)
    assert (err <= 20 * rel * (mag + np.abs(want)) + (F16_REL * np.abs(want) * 1.001 + 2.0 ** -25 if half else 0) + 1e-30).all()
    assert (got[pos.numpy() < 0] == 0).all()


def run(q, pos, pages, c, **kw):
    from webpytorch_amd import core
    return core.paged_attention(q.cuda(), pos.cuda(), pages.cuda(), c.cuda(), **kw)


TYPES = [("float32", "float16"), ("float16", "float16"), ("float32", "float32"), ("float16", "float32")]


@pytest.mark.parametrize("x,cache", TYPES)
@pytest.mark.parametrize("NH,NKV,HD", [(2, 2, 64), (14, 2, 64), (4, 1, 128), (7, 1, 128), (3, 3, 192), (8, 2, 256), (20, 1, 64)])
@pytest.mark.parametrize("T", [1, 2, 5])
def test_heads_types_and_lengths(gpu, NH, NKV, HD, T, x, cache):
    import torch
    lens = [1, 0, 15, 16, 17, 31, 32, 33, 64, 100, 255, 257, 300]
    a = setup(torch, HD + T, lens, T, NH, NKV, HD, 16, x, cache)
    check(run(*a), *a)


@pytest.mark.parametrize("x,cache", TYPES)
@pytest.mark.parametrize("P", [16, 32, 64, 256, 4096])
def test_page_sizes(gpu, P, x, cache):
    import torch
    a = setup(torch, P, [P - 1, P, P + 1, 3 * P + 7, 1], 2, 4, 2, 64, P, x, cache)
    check(run(*a), *a)


@pytest.mark.parametrize("x,cache", TYPES)
@pytest.mark.parametrize("NH,NKV,HD,T", [(4, 2, 64, 9), (8, 1, 64, 8), (4, 1, 64, 33), (7, 1, 128, 5), (4, 1, 128, 9), (8, 1, 128, 6), (6, 2, 192, 7),
                                         (8, 2, 256, 5), (2, 1, 128, 70)])
def test_several_rows(gpu, NH, NKV, HD, T, x, cache):
    """Several tiles of rows, several workgroups of tiles."""
    import torch
    a = setup(torch, T, [T, T + 40, 500, 3], T, NH, NKV, HD, 32, x, cache)
    check(run(*a), *a)


@pytest.mark.parametrize("x,cache", TYPES)
@pytest.mark.parametrize("S,NH,NKV,HD,longest", [(1, 4, 1, 128, 9000), (1, 14, 2, 64, 20000), (3, 8, 2, 256, 5000), (2, 4, 2, 192, 7001)])
def test_long_sequences_are_split_and_joined(gpu, S, NH, NKV, HD, longest, x, cache):
    import torch
    from webpytorch_amd import core, _lib
    lens = [longest, 0, 700][:S]
    a = setup(torch, S, lens, 2, NH, NKV, HD, 64, x, cache)
    code = _lib.MIQ_F16 if cache == "float16" else _lib.MIQ_F32
    assert core.paged_attention_workspace_bytes(S, 2, NH, NKV, HD, 64, a[2].shape[1], code) > 0
    check(run(*a), *a)


@pytest.mark.parametrize("S", [63, 64, 65, 130, 700])
@pytest.mark.parametrize("T", [1, 3])
def test_many_sequences(gpu, S, T):
    """Sequences from 64 on are looked up in several rounds; long ones among short ones."""
    import torch
    g = torch.Generator().manual_seed(S)
    lens = torch.randint(0, 60, (S,), generator=g).tolist()
    lens[S // 2] = 3000
    lens[-1] = 1000
    a = setup(torch, S, lens, T, 4, 2, 64, 16, "float32", "float16")
    check(run(*a), *a)


@pytest.mark.parametrize("cache", ["float16", "float32"])
def test_tokens_of_other_orders(gpu, cache):
    """Positions that are not in order, missing ones between them, past the table, and one sequence without any."""
    import torch
    q, pos, pages, c = setup(torch, 8, [200, 90, 64], 5, 4, 2, 64, 32, "float32", cache)
    c = torch.nan_to_num(c)
    pos = torch.tensor([[150, -1, 3, 199, 0], [-1] * 5, [63, 2000, 5, -7, 2 ** 31 - 1]], dtype=torch.int32)
    check(run(q, pos, pages, c), q, pos, pages, c)


@pytest.mark.parametrize("cache", ["float16", "float32"])
@pytest.mark.parametrize("P", [16, 32])
def test_missing_pages_are_left_out(gpu, cache, P):
    import torch
    q, pos, pages, c = setup(torch, 9, [10 * P + 3, 4 * P, 2 * P, 9 * P], 2, 4, 2, 128, P, "float32", cache)
    pages[0, 2], pages[0, 5] = -1, c.shape[0]     # outside the cache on both sides
    pages[1, :], pages[2, 1] = -5, 2 ** 31 - 1    # a sequence with nothing left
    pages[3, -1] = -1
    out = run(q, pos, pages, c)
    check(out, q, pos, pages, c)
    assert (out[1] == 0).all()


@pytest.mark.parametrize("x,cache", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_non_finite_values_reach_their_tokens_alone(gpu, bad, x, cache):
    """Position n's value is seen by the tokens from n on, in its dimension; an earlier key that is NaN by all after it."""
    import torch
    T, n = 4, 300
    q, pos, pages, c = setup(torch, 4, [n, 50], T, 8, 2, 64, 32, x, cache)
    clean = run(q, pos, pages, c)
    at = pages[0, (n - 2) // 32], (n - 2) % 32
    c[at[0], 1, 0, at[1], 7] = bad  # of kv head 0, dimension 7: tokens 2 and 3 of heads 0 .. 3
    out = run(q, pos, pages, c)
    hit = torch.zeros(out.shape, dtype=torch.bool)
    hit[0, 2:, :4, 7] = True
    assert not torch.isfinite(out.cpu()[hit]).any() and torch.equal(out.cpu()[~hit], clean.cpu()[~hit])
    c[at[0], 1, 0, at[1], 7] = 0
    c[at[0], 0, 1, at[1], 3] = float("nan")  # a key of kv head 1
    out = run(q, pos, pages, c)
    hit = torch.zeros(out.shape, dtype=torch.bool)
    hit[0, 2:, 4:] = True
    assert torch.isnan(out.cpu()[hit]).all() and torch.isfinite(out.cpu()[~hit]).all()


@pytest.mark.parametrize("x,cache", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-3, 30.0])
def test_scales(gpu, scale, x, cache):
    import torch
    a = setup(torch, 6, [500, 40], 2, 4, 2, 64, 16, x, cache)
    # scores of up to 30 x 40: a relative error of 2^-22 of them is one of e^(1200 2^-22) - 1 = 3e-4 in a probability
    check(run(*a, scale=scale), *a, scale=scale, rel=F32_REL if abs(scale) < 1 else 3e-4)


@pytest.mark.parametrize("size", [2.0 ** -40, 2.0 ** -120, 2.0 ** 30])
def test_queries_of_any_size(gpu, size):
    """fp32 rows keep their low bits in the fp16 products, with the scale taken off again."""
    import torch
    q, pos, pages, c = setup(torch, 7, [400, 33], 2, 4, 1, 128, 32, "float32", "float16")
    check(run(q * size, pos, pages, c, scale=128 ** -0.5 / size), q, pos, pages, c)


@pytest.mark.parametrize("x,cache", TYPES)
def test_one_sharp_score_and_growing_scores(gpu, x, cache):
    """One key beside thousands of small ones; scores that grow with the position (the reference is raised again and again)."""
    import torch
    n, HD = 3000, 64
    q, pos, pages, c = setup(torch, 5, [n], 1, 2, 1, HD, 32, x, cache)
    table = pages[0].long()
    q[:] = 0
    q[..., 0] = 1.0
    for kind in ("sharp", "up", "down"):
        ramp = torch.zeros(n) if kind == "sharp" else torch.arange(n) * (0.02 if kind == "up" else -0.02)
        if kind == "sharp":
            ramp[1234] = 9.0
        k = torch.zeros(table.numel() * 32)
        k[:n] = ramp
        c[table, 0, 0, :, 0] = k.view(-1, 32).to(c.dtype)
        check(run(q, pos, pages, c, scale=1.0), q, pos, pages, c, scale=1.0)


def test_replays_match_the_eager_call(gpu):
    """A captured append and attention, replayed as positions move on, with eager calls between the replays."""
    import torch
    from webpytorch_amd import core
    q, pos, pages, c = setup(torch, 3, [2900, 40, 700], 1, 4, 2, 64, 16, "float32", "float16", extra=40)
    c = torch.nan_to_num(c).cuda()
    pages = torch.cat([pages, torch.full((3, 4), -1, dtype=torch.int32)], 1)
    free = [p for p in range(c.shape[0]) if p not in pages.flatten().tolist()]
    for s in range(3):
        n = int((pages[s] >= 0).sum())
        pages[s, n:n + 3] = torch.tensor(free[3 * s:3 * s + 3], dtype=torch.int32)
    pages, pos = pages.cuda(), pos.cuda()
    r = core.rope_tables(4000, 64)
    qkv = torch.randn((3, 1, 8 * 64), device="cuda")
    step = lambda: core.paged_attention(core.paged_append(qkv, pos, pages, c, 4, r), pos, pages, c)  # noqa: E731
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(6):
        qkv.copy_(torch.randn((3, 1, 8 * 64), device="cuda"))
        pos += 1
        before = c.clone()
        g.replay()
        torch.cuda.synchronize()
        got, after = out.clone(), c.clone()
        c.copy_(before)
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(after, c), i


def test_two_graphs_and_two_streams(gpu):
    """Two captured calls replayed at a time, and eager calls on two streams, each with its own workspace."""
    import torch
    from webpytorch_amd import core
    sets = [[t.cuda() for t in setup(torch, i, [6000 + 1000 * i, 50], 1, 4, 2, 64, 32, "float32", "float16")] for i in range(2)]
    alone = [core.paged_attention(*s) for s in sets]
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            outs.append(core.paged_attention(*s))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(alone, outs))
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    for _ in range(20):
        for st, s, a in zip(streams, sets, alone):
            with torch.cuda.stream(st):
                wrong += 0 if torch.cuda.is_current_stream_capturing() else (core.paged_attention(*s) != a).sum()
        torch.cuda.synchronize()
    assert int(wrong) == 0


def test_two_threads_on_one_stream(gpu):
    import torch
    from webpytorch_amd import core
    sets = [[t.cuda() for t in setup(torch, i, [5000 + 900 * i], 1, 4, 2, 64, 32, "float32", "float16")] for i in range(2)]
    alone = [core.paged_attention(*s) for s in sets]
    wrong = [torch.zeros((), dtype=torch.int64, device="cuda") for _ in sets]
    errors, start = [], threading.Barrier(2)

    def work(i):
        try:
            start.wait(30)
            for _ in range(50):
                wrong[i] += (core.paged_attention(*sets[i]) != alone[i]).sum()
        except Exception as e:  # reported by the test's own thread
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    torch.cuda.synchronize()
    assert not errors, errors
    assert [int(w) for w in wrong] == [0, 0]


def test_far_pages(gpu):
    """A cache of more than 2^32 values: pages at its end are written and read where they are."""
    import torch
    from webpytorch_amd import core
    NKV, P, HD = 8, 256, 128
    num = (1 << 32) // (2 * NKV * P * HD) + 3
    c = torch.zeros((num, 2, NKV, P, HD), dtype=torch.float16, device="cuda")
    pages = torch.tensor([[num - 1, num - 2]], dtype=torch.int32).cuda()
    n = 300
    qkv = torch.randn((1, n, (NKV * 4 + 2 * NKV) * HD)).cuda()
    pos = torch.arange(n, dtype=torch.int32).cuda()[None]
    q = core.paged_append(qkv, pos, pages, c, NKV * 4)
    small = c[num - 2:].clone()
    assert not (small[1] == 0).all() and (c[:2] == 0).all()
    near = torch.tensor([[1, 0]], dtype=torch.int32).cuda()
    a, b = core.paged_attention(q[:, -1:], pos[:, -1:], pages, c), core.paged_attention(q[:, -1:], pos[:, -1:], near, small)
    assert torch.equal(a, b)
    check(a, q[:, -1:].cpu(), pos[:, -1:].cpu(), near.cpu(), small.cpu())


def test_out_is_written_and_the_rest_left(gpu):
    import torch
    from webpytorch_amd import core
    q, pos, pages, c = (t.cuda() for t in setup(torch, 2, [40, 500], 2, 4, 2, 64, 16, "float16", "float16"))
    buf = torch.full((q.numel() + 64,), 3.0, dtype=torch.float16, device="cuda")
    out = buf[32:-32].view(q.shape)
    core.paged_attention(q, pos, pages, c, out=out)
    assert torch.equal(out, core.paged_attention(q, pos, pages, c)) and (buf[:32] == 3).all() and (buf[-32:] == 3).all()
    wide = torch.randn((2, 2, 4, 128), device="cuda", dtype=torch.float16)[..., :64]  # rows that are not contiguous
    assert torch.equal(core.paged_attention(wide, pos, pages, c), core.paged_attention(wide.contiguous(), pos, pages, c))
    with pytest.raises(ValueError, match="apart"):
        core.paged_attention(q, pos, pages, c, out=q)
