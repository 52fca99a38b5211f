"""GPU: the calls of a batch's serving as programs make them: captured at the largest sizes, two graphs and two threads at a time, long
prompts, caches shared by sequences, outputs handed in."""
import threading

import numpy as np
import pytest

from oracle import paged
from test_gpu_paged import check, run, setup
from test_gpu_verify import rows

pytestmark = pytest.mark.gpu


def replay(call, change, n=4):
    """The call captured, then replayed with other inputs and eager calls between: every replay is the eager call's."""
    import torch
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for i in range(n):
        change(i)
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


@pytest.mark.parametrize("S,D,V", [(5000, 2, 60), (9000, 0, 40), (600, 3, 9000)])
def test_captured_verification_of_many_sequences(gpu, S, D, V):
    import torch
    from webpytorch_amd import core
    g = torch.Generator(device="cuda").manual_seed(S)
    x = torch.randn((S, D + 1, V), device="cuda", generator=g) * 2
    ids = torch.randint(0, V, (S, D), device="cuda", generator=g, dtype=torch.int32)
    u = torch.rand((S, D + 1), device="cuda", generator=g)
    replay(lambda: core.verify_drafts(x, ids, u), lambda i: u.copy_(torch.rand(u.shape, device="cuda", generator=g)))
    some = slice(S - 200, S)
    got = core.verify_drafts(x, ids, u)
    tokens, accepted, near = paged.verify(x[some].cpu().numpy(), ids[some].cpu().numpy(), u[some].cpu().numpy())
    sure = near > 1e-11
    np.testing.assert_array_equal(got.accepted[some].cpu().numpy(), accepted)
    np.testing.assert_array_equal(got.tokens[some].cpu().numpy()[sure], tokens[sure])


def test_captured_attention_at_the_most_counters(gpu):
    """As many sequences and heads as are split: the last ones' counters are cleared too."""
    import torch
    from webpytorch_amd import core
    lens = [20] * 512
    lens[0], lens[300], lens[511] = 3000, 2500, 4000
    q, pos, pages, c = setup(torch, 1, lens, 1, 8, 8, 64, 16, "float16", "float16")
    c = torch.nan_to_num(c)
    q, pos, pages, c = (t.cuda() for t in (q, pos, pages, c))
    replay(lambda: [core.paged_attention(q, pos, pages, c)], lambda i: q.copy_(torch.randn(q.shape, device="cuda").to(q.dtype)))
    some = [0, 1, 300, 510, 511]
    check(core.paged_attention(q, pos, pages, c)[some], q[some].cpu(), pos[some].cpu(), pages[some].cpu(), c.cpu())


def test_two_verifications_at_a_time(gpu):
    """Two graphs on two streams, then two threads on one stream."""
    import torch
    from webpytorch_amd import core
    sets = [[torch.from_numpy(a).cuda() for a in rows(20 + i, 3 + i, 2, 30000, np.float32)] for i in range(2)]
    call = lambda s: core.verify_drafts(s[0], s[2], s[3], s[1])  # noqa: E731
    alone = [call(s) for s in sets]
    graphs, outs = [], []
    for s in sets:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(s))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o, w in zip(outs, alone) for a, b in zip(o, w))
    wrong = [torch.zeros((), dtype=torch.int64, device="cuda") for _ in sets]
    errors, start = [], threading.Barrier(2)

    def work(i):
        try:
            start.wait(30)
            for _ in range(50):
                wrong[i] += (call(sets[i]).tokens != alone[i].tokens).sum()
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


@pytest.mark.parametrize("x,cache", [("float32", "float16"), ("float16", "float32")])
def test_a_prompt_through_the_cache(gpu, x, cache):
    """Hundreds of tokens of a sequence at once, behind others: every row of every tile."""
    import torch
    a = setup(torch, 12, [420, 333], 330, 4, 2, 128, 32, x, cache)
    check(run(*a), *a)


def test_shared_pages(gpu):
    """Two sequences with one prefix share its pages; each has its own behind them."""
    import torch
    from webpytorch_amd import core
    q, pos, pages, c = setup(torch, 13, [100, 96], 1, 4, 2, 64, 16, "float32", "float16")
    c = torch.nan_to_num(c)
    pages[1, :6] = pages[0, :6]
    check(run(q, pos, pages, c), q, pos, pages, c)
    dev = c.cuda()
    before = dev.clone()
    qkv = torch.randn((2, 1, 8 * 64)).cuda()
    pos2 = torch.tensor([[100], [96]], dtype=torch.int32)
    pages = torch.cat([pages, torch.full((2, 1), -1, dtype=torch.int32)], 1)
    used = set(pages.flatten().tolist())
    pages[1, 6] = next(p for p in range(c.shape[0]) if p not in used)
    core.paged_append(qkv, pos2.cuda(), pages.cuda(), dev, 4)
    shared = pages[0, :6].long()
    assert torch.equal(dev[shared], before[shared])
    v = qkv.view(2, 8, 64)[:, 6:].half()
    assert torch.equal(dev[pages[0, 6].item(), 1, :, 4], v[0]) and torch.equal(dev[pages[1, 6].item(), 1, :, 0], v[1])


def test_outputs_handed_in(gpu):
    import torch
    from webpytorch_amd import core
    q, pos, pages, c = (t.cuda() for t in setup(torch, 14, [40, 70], 2, 4, 2, 64, 16, "float32", "float32"))
    c = torch.nan_to_num(c)
    qkv = torch.randn((2, 2, 8 * 64), device="cuda")
    r = core.rope_tables(100, 64)
    a, b = c.clone(), c.clone()
    out = torch.full((2, 2, 4, 64), 7.0, device="cuda")
    assert core.paged_append(qkv, pos, pages, a, 4, r, out=out) is out
    assert torch.equal(out, core.paged_append(qkv, pos, pages, b, 4, r)) and torch.equal(a, b)
    with pytest.raises(ValueError, match="apart"):
        core.paged_append(qkv, pos, pages, a, 4, r, out=qkv.view(-1)[:2 * 2 * 4 * 64])
    with pytest.raises(ValueError, match="out is a contiguous"):
        core.paged_append(qkv, pos, pages, a, 4, r, out=out[:1])
    x = torch.randn((6, 4, 64), device="cuda")
    p = torch.arange(6, dtype=torch.int32, device="cuda")
    want = core.rope(x, p, r)
    assert core.rope(x, p, r, out=x) is x and torch.equal(x, want)
    with pytest.raises(ValueError, match="lie apart"):
        core.rope(x[:3], p[:3], r, out=x.view(-1)[64:64 + 3 * 256].view(3, 4, 64))


@pytest.mark.parametrize("call,exc,text", [
    (lambda c, t: c.rope(t.zeros((2, 3, 64), device="cuda"), t.zeros(3, dtype=t.int32, device="cuda"), c.rope_tables(8, 64)), ValueError, "positions"),
    (lambda c, t: c.rope(t.zeros((2, 3, 64), device="cuda"), t.zeros(2, dtype=t.int64, device="cuda"), c.rope_tables(8, 64)), TypeError, "positions"),
    (lambda c, t: c.rope(t.zeros((2, 3, 64), device="cuda"), t.zeros(2, dtype=t.int32, device="cuda"), c.rope_tables(8, 66)), ValueError, "rot at most 64"),
    (lambda c, t: c.rope(t.zeros((2, 3, 64), device="cuda", dtype=t.bfloat16), t.zeros(2, dtype=t.int32, device="cuda"), c.rope_tables(8, 64)), TypeError, "bfloat16"),
    (lambda c, t: c.paged_append(t.zeros((1, 2, 255), device="cuda"), t.zeros((1, 2), dtype=t.int32, device="cuda"),
                                 t.zeros((1, 1), dtype=t.int32, device="cuda"), c.paged_cache(2, 1, 16, 64), 2), ValueError, "255 values"),
    (lambda c, t: c.paged_append(t.zeros((1, 2, 256), device="cuda"), t.zeros((2, 1), dtype=t.int32, device="cuda"),
                                 t.zeros((2, 1), dtype=t.int32, device="cuda"), c.paged_cache(2, 1, 16, 64), 2), ValueError, "positions"),
    (lambda c, t: c.paged_attention(t.zeros((1, 2, 2, 64), device="cuda"), t.zeros((1, 2), dtype=t.int32, device="cuda"),
                                    t.zeros((2, 1), dtype=t.int32, device="cuda"), c.paged_cache(2, 1, 16, 64)), ValueError, "pages of 2"),
    (lambda c, t: c.paged_attention(t.zeros((1, 2, 3, 64), device="cuda"), t.zeros((1, 2), dtype=t.int32, device="cuda"),
                                    t.zeros((1, 1), dtype=t.int32, device="cuda"), c.paged_cache(2, 2, 16, 64)), ValueError, "does not go"),
    (lambda c, t: c.paged_attention(t.zeros((1, 2, 2, 64), device="cuda"), t.zeros((1, 2), dtype=t.int32, device="cuda"),
                                    t.zeros((1, 1), dtype=t.int32, device="cuda"), c.paged_cache(2, 1, 16, 64)[:, :, :, ::2]), ValueError, "page"),
    (lambda c, t: c.verify_drafts(t.zeros((2, 3, 9), device="cuda"), t.zeros((2, 3), dtype=t.int32, device="cuda"), t.zeros((2, 3), device="cuda")),
     ValueError, "drafts"),
    (lambda c, t: c.verify_drafts(t.zeros((2, 3, 9), device="cuda"), t.zeros((2, 2), dtype=t.int32, device="cuda"), t.zeros((2, 2), device="cuda")),
     ValueError, "uniforms"),
    (lambda c, t: c.verify_drafts(t.zeros((2, 3, 9), device="cuda"), t.zeros((2, 2), dtype=t.int32, device="cuda"), t.zeros((2, 3), device="cuda"),
                                  t.zeros((2, 2, 9), device="cuda", dtype=t.float16)), TypeError, "draft_logits"),
    (lambda c, t: c.verify_drafts(t.zeros((2, 3, 9), device="cuda"), t.zeros((2, 2), dtype=t.int32, device="cuda"), t.zeros((2, 3), device="cuda"),
                                  temperature=-1.0), ValueError, "temperature")])
def test_refusals(gpu, call, exc, text):
    import torch
    from webpytorch_amd import core
    with pytest.raises(exc, match=text):
        call(core, torch)


def test_empty_batches(gpu):
    import torch
    from webpytorch_amd import core
    c = core.paged_cache(2, 1, 16, 64)
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    z = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    assert core.rope(z(0, 2, 64), i(0), core.rope_tables(4, 64)).shape == (0, 2, 64)
    assert core.paged_append(z(0, 3, 256), i(0, 3), i(0, 2), c, 2).shape == (0, 3, 2, 64)
    assert core.paged_append(z(2, 0, 256), i(2, 0), i(2, 2), c, 2).shape == (2, 0, 2, 64)
    assert core.paged_attention(z(2, 0, 2, 64), i(2, 0), i(2, 2), c).shape == (2, 0, 2, 64)
    assert (core.paged_attention(z(2, 1, 2, 64) + 1, i(2, 1), i(2, 0), c) == 0).all()  # no pages at all
    assert (core.paged_append(z(2, 1, 256) + 1, i(2, 1), i(2, 0), c, 2) == 0).all() and (c == 0).all()
    assert core.verify_drafts(z(0, 2, 9), i(0, 1), z(0, 2)).tokens.shape == (0, 2)
