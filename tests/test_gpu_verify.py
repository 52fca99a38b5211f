"""GPU: verification of drafted tokens, and a batch served with all of it, against float64 (`oracle/paged.py`)."""
import math

import numpy as np
import pytest

from oracle import paged

pytestmark = pytest.mark.gpu

# The kernel's probabilities are off by 3e-13 (2.2e-13 of the series, the rest of fp64 sums): a draw this near to a border between
# tokens may fall on either side. No seed below comes near it (checked).
BORDER = 1e-11


def rows(seed, S, D, V, dt, peak=3.0):
    g = np.random.default_rng(seed)
    x = (g.standard_normal((S, D + 1, V)) * g.uniform(0.5, peak, (S, D + 1, 1))).astype(dt)
    d = (x[:, :D] + 0.5 * g.standard_normal((S, D, V))).astype(dt)
    ids = np.zeros((S, D), np.int32)
    for s in range(S):
        for i in range(D):
            ids[s, i] = g.choice(V, p=paged.law(d[s, i], 1.0))
    return x, d, ids, g.random((S, D + 1)).astype(np.float32)


def check(x, ids, u, d=None, temperature=1.0):
    import torch
    from webpytorch_amd import core
    dev = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    t = dev(temperature) if isinstance(temperature, np.ndarray) else temperature
    got = core.verify_drafts(dev(x), dev(ids), dev(u), dev(d), temperature=t)
    tokens, accepted, near = paged.verify(x, ids, u, d, temperature)
    assert near.min() > BORDER
    assert got.tokens.dtype == torch.int32 and got.accepted.dtype == torch.int32
    np.testing.assert_array_equal(got.accepted.cpu().numpy(), accepted)
    np.testing.assert_array_equal(got.tokens.cpu().numpy(), tokens)
    return tokens, accepted


@pytest.mark.parametrize("dt", [np.float32, np.float16])
@pytest.mark.parametrize("S,D,V", [(1, 4, 1000), (5, 3, 4095), (3, 2, 4096), (3, 2, 4097), (2, 1, 32003), (40, 5, 257), (1, 0, 5000), (3, 32, 50),
                                   (2, 2, 1), (9, 3, 2), (7, 4, 17), (1, 6, 151936)])
def test_drawn_drafts(gpu, S, D, V, dt):
    x, d, ids, u = rows(S * 100 + D, S, D, V, dt)
    check(x, ids, u, d)
    check(x, ids, u, d, temperature=0.6)
    check(x, ids, u)


def test_every_outcome_occurs(gpu):
    x, d, ids, u = rows(1, 64, 4, 300, np.float32)
    _, accepted = check(x, ids, u, d)
    assert set(accepted.tolist()) == {0, 1, 2, 3, 4}
    _, accepted = check(x, np.argmax(x[:, :4], -1).astype(np.int32), u)
    assert len(set(accepted.tolist())) > 2


@pytest.mark.parametrize("dt", [np.float32, np.float16])
def test_greedy(gpu, dt):
    """Temperature 0: the lowest index of the largest logit, NaN as -inf; some drafts agree."""
    g = np.random.default_rng(2)
    x = np.round(g.standard_normal((12, 4, 9000)) * 2).astype(dt)  # many equal ones
    ids = np.argmax(x[:, :3], -1).astype(np.int32)
    ids[::3, 1] += 1
    ids[1, 0] = -1
    x[4, 0, :50] = np.nan
    x[5, 0, :] = -np.inf
    x[6, 0, 77], x[6, 0, 8000] = np.inf, np.inf
    x[7, 3] = np.nan
    u = g.random((12, 4)).astype(np.float32)
    tokens, _ = check(x, ids, u, temperature=0.0)
    assert tokens[5, 0] == -1
    d = g.standard_normal((12, 3, 9000)).astype(dt)
    np.testing.assert_array_equal(check(x, ids, u, d, temperature=0.0)[0], tokens)


def test_temperatures_of_sequences(gpu):
    x, d, ids, u = rows(3, 9, 3, 500, np.float32)
    t = np.array([0.0, 0.3, 1.0, 2.5, 1e-3, 0.0, 100.0, 0.7, 1.3], np.float32)
    check(x, ids, u, d, temperature=t)
    check(x, ids, u, temperature=t)


def test_fewer_drafts_and_ids_outside_the_vocabulary(gpu):
    x, d, ids, u = rows(4, 8, 4, 600, np.float32)
    ids[0, 0] = ids[1, 1] = ids[2, 3] = -1
    ids[3] = -1
    ids[4, 0], ids[5, 2], ids[6, 1] = 600, 2 ** 31 - 1, 599
    check(x, ids, u, d)
    check(x, ids, u)


def test_masked_and_non_finite_logits(gpu):
    x, d, ids, u = rows(5, 10, 2, 3000, np.float32)
    g = np.random.default_rng(9)
    x[:, :, g.random(3000) < 0.7] = -np.inf
    d[1, 0, :2990] = -np.inf
    x[2, 0, 5] = np.nan      # no distribution: nothing accepted, no token
    x[3, 0, 5] = np.inf
    x[4, 0] = -np.inf
    x[5, 2] = -np.inf        # behind the last draft
    d[6, 0, 9] = np.nan      # a draft's row without one: refused, drawn from the target
    d[7, 1] = -np.inf
    x[8, 0] = -np.inf
    x[8, 0, 42] = 0.0        # one token alone
    ids[8, 0] = 42
    tokens, accepted = check(x, ids, u, d)
    assert (accepted[[2, 3, 4, 6]] == 0).all() and (tokens[[2, 3, 4], 0] == -1).all() and tokens[6, 0] >= 0
    check(x, ids, u)


def test_extremes_of_the_random_numbers(gpu):
    """0 and the largest number below 1, at draws and acceptances."""
    x, d, ids, u = rows(6, 6, 2, 5000, np.float32)
    x[:, :, :3] = -np.inf
    x[:, :, -2:] = -np.inf
    for v in (0.0, 1.0 - 2.0 ** -24):
        u[:] = v
        import torch
        from webpytorch_amd import core
        for dd in (d, None):
            got = core.verify_drafts(*(torch.from_numpy(a).cuda() for a in (x, ids, u)), None if dd is None else torch.from_numpy(dd).cuda())
            tokens, accepted, near = paged.verify(x, ids, u, dd)
            np.testing.assert_array_equal(got.accepted.cpu().numpy(), accepted)
            sure = (near > BORDER) | (v == 0.0)  # at 0 the border is the start itself
            np.testing.assert_array_equal(got.tokens.cpu().numpy()[sure], tokens[sure])


def test_the_draft_is_the_target(gpu):
    """The same rows: everything is accepted. The draft's only alternative gone: the draft is the answer even if refused."""
    x, d, ids, u = rows(7, 5, 3, 400, np.float32)
    _, accepted = check(x, ids, u, x[:, :3].copy())
    assert (accepted == 3).all()
    import torch
    from webpytorch_amd import core
    one = np.full((1, 2, 50), -np.inf, np.float32)
    one[:, :, 7] = 1.0
    got = core.verify_drafts(*(torch.from_numpy(a).cuda() for a in (one, np.array([[7]], np.int32), np.array([[1.0, 0.5]], np.float32))))
    assert got.accepted.item() == 0 and got.tokens.tolist() == [[7, -1]]


@pytest.mark.parametrize("dt", [np.float32, np.float16])
def test_padded_and_unaligned_rows(gpu, dt):
    import torch
    from webpytorch_amd import core
    x, d, ids, u = rows(8, 4, 3, 999, dt)
    want = paged.verify(x, ids, u, d)
    t = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    buf = torch.full((4, 5, 1041), 9.0, dtype=t(x).dtype, device="cuda")
    buf[:, 1:, 1:1000] = t(x)
    db = torch.full((3, 4, 1024), 9.0, dtype=t(x).dtype, device="cuda")
    db[:, :, :999] = t(d).transpose(0, 1)
    got = core.verify_drafts(buf[:, 1:, 1:1000], t(ids), t(u), db[:, :, :999].transpose(0, 1))
    np.testing.assert_array_equal(got.tokens.cpu().numpy(), want[0])
    turned = t(x).permute(2, 0, 1).contiguous().permute(1, 2, 0)
    got = core.verify_drafts(turned, t(ids), t(u), t(d))
    np.testing.assert_array_equal(got.tokens.cpu().numpy(), want[0])


def test_long_rows(gpu):
    """More chunks than sums are kept of: several rounds of logits a sum."""
    import torch
    from webpytorch_amd import core
    V = 4096 * 1024 + 4097 * 3
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((2, 2, V), device="cuda", generator=g)
    ids = torch.tensor([[5], [V - 1]], dtype=torch.int32).cuda()
    u = torch.tensor([[0.9, 0.25], [0.9, 0.999]], device="cuda")
    got = core.verify_drafts(x, ids, u)
    tokens, accepted, near = paged.verify(x.cpu().numpy(), ids.cpu().numpy(), u.cpu().numpy())
    assert near.min() > BORDER
    np.testing.assert_array_equal(got.tokens.cpu().numpy(), tokens)


def test_tokens_are_distributed_as_the_target(gpu):
    """First tokens over many random numbers: the target's probabilities, whatever the draft's are (5 standard deviations)."""
    import torch
    from webpytorch_amd import core
    V, S, N = 12, 4096, 4
    g = torch.Generator(device="cuda").manual_seed(1)
    x, d = (torch.randn((1, n, V), device="cuda", generator=g) * 1.5 for n in (2, 1))
    p, q = (torch.softmax(t[0, 0].double(), 0) for t in (x, d))
    count = torch.zeros(V, dtype=torch.float64, device="cuda")
    for _ in range(N):
        ids = torch.multinomial(q, S, replacement=True, generator=g).to(torch.int32)[:, None]
        u = torch.rand((S, 2), device="cuda", generator=g)
        r = core.verify_drafts(x.expand(S, 2, V), ids, u, d.expand(S, 1, V))
        count += torch.bincount(r.tokens[:, 0].long(), minlength=V)
    n = S * N
    assert ((count - n * p).abs() < 5 * (n * p * (1 - p)).sqrt() + 1).all()


def test_replays(gpu):
    import torch
    from webpytorch_amd import core
    x, d, ids, u = (torch.from_numpy(a).cuda() for a in rows(10, 6, 3, 20000, np.float32))
    core.verify_drafts(x, ids, u, d)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = core.verify_drafts(x, ids, u, d)
    for _ in range(5):
        u.copy_(torch.rand_like(u))
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in r]
        want = core.verify_drafts(x, ids, u, d)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_batch_served_with_drafts(gpu):
    """Three sequences through one attention layer and a head: prompts appended in one padded batch, then steps of three drafted
    tokens each from the paged cache (pages handed out as sequences grow, refused drafts overwritten by the next step), tokens
    verified. Every step's logits against float64 over the sequence so far without a cache, its tokens against float64's verdict."""
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(4)
    S, NH, NKV, HD, P, V, D = 3, 4, 2, 64, 16, 300, 3
    H, W = NH * HD, (NH + 2 * NKV) * HD
    emb, wqkv, head = torch.randn((V, H), generator=g), torch.randn((H, W), generator=g) / 16, torch.randn((H, V), generator=g) / 4
    qn, kn = (1 + 0.2 * torch.randn(HD, generator=g) for _ in range(2))
    r = core.rope_tables(200, 32, scaling={"rope_type": "linear", "factor": 2.0}, interleaved=True)
    cache = core.paged_cache(24, NKV, P, HD, torch.float32)
    cache.fill_(float("nan"))
    pages, free = torch.full((S, 8), -1, dtype=torch.int32), list(range(23, -1, -1))
    dev = [t.cuda() for t in (emb, wqkv, head, qn, kn)]

    def forward(tokens, pos):
        """Logits (S, T, V) of tokens at positions, through the cache."""
        for s in range(S):  # pages for the positions
            for n in range((int(pos[s].max()) + P) // P):
                if pages[s, n] < 0:
                    pages[s, n] = free.pop()
        qkv = (dev[0][tokens.cuda().clamp(min=0).long()].double() @ dev[1].double()).float()
        p, t = pos.cuda(), pages.cuda()
        q = core.paged_append(qkv, p, t, cache, NH, r, qn=dev[3], kn=dev[4])
        a = core.paged_attention(q, p, t, cache)
        return (a.flatten(2).double() @ dev[2].double()).float()

    cs, sn = r.cos.double().cpu().numpy(), r.sin.double().cpu().numpy()

    def plain(seq):
        """float64 logits of every position of a text."""
        x = (emb[seq].double() @ wqkv.double()).numpy().reshape(len(seq), NH + 2 * NKV, HD)
        rms = lambda y, w: y / np.sqrt((y * y).mean(-1, keepdims=True) + 1e-6) * w.double().numpy()  # noqa: E731
        at = np.arange(len(seq))
        q, _ = paged.rope(rms(x[:, :NH], qn), at, cs, sn, True)
        k, _ = paged.rope(rms(x[:, NH:NH + NKV], kn), at, cs, sn, True)
        out = np.zeros((len(seq), NH, HD))
        for h in range(NH):
            a = q[:, h] @ k[:, h // 2].T / math.sqrt(HD)
            a = np.where(at[None, :] > at[:, None], -np.inf, a)
            e = np.exp(a - a.max(-1, keepdims=True))
            out[:, h] = e / e.sum(-1, keepdims=True) @ x[:, NH + NKV + h // 2]
        return out.reshape(len(seq), -1) @ head.double().numpy()

    texts = [torch.randint(0, V, (n,), generator=g).tolist() for n in (5, 17, 40)]
    T = max(map(len, texts))
    ids, pos = torch.full((S, T), -1, dtype=torch.int32), torch.full((S, T), -1, dtype=torch.int32)
    for s, t in enumerate(texts):
        ids[s, :len(t) - 1], pos[s, :len(t) - 1] = torch.tensor(t[:-1], dtype=torch.int32), torch.arange(len(t) - 1, dtype=torch.int32)
    forward(ids, pos)
    counts = set()
    for step in range(12):
        drafts = torch.full((S, D), -1, dtype=torch.int32)
        for s, t in enumerate(texts):  # drafts: the likely token, or any; the second sequence has fewer
            for i in range(D - (s == 1)):
                lg = plain(t + drafts[s, :i].tolist())[-1]
                drafts[s, i] = int(lg.argmax()) if torch.rand((), generator=g) < 0.8 else int(torch.randint(0, V, (), generator=g))
        ids = torch.cat([torch.tensor([[t[-1]] for t in texts], dtype=torch.int32), drafts], 1)
        pos = torch.tensor([[len(t) - 1] for t in texts], dtype=torch.int32) + torch.arange(D + 1, dtype=torch.int32)[None]
        pos[ids < 0] = -1
        u = torch.rand((S, D + 1), generator=g)
        lg = forward(ids, pos)
        verdict = core.verify_drafts(lg, drafts.cuda(), u.cuda(), temperature=0.3)
        for s, t in enumerate(texts):
            n = int((ids[s] >= 0).sum())
            want = plain(t + drafts[s, :n - 1].tolist())[-n:]
            err = np.abs(lg[s, :n].double().cpu().numpy() - want).max()
            assert err < 2e-5 * np.abs(want).max(), (step, s, err)  # 128 fp32 sums of cache rows, products and softmax: 2^-24 each
        tokens, accepted, near = paged.verify(lg.cpu().numpy(), drafts.numpy(), u.numpy(), None, 0.3)
        assert near.min() > BORDER
        np.testing.assert_array_equal(verdict.tokens.cpu().numpy(), tokens)
        for s in range(S):
            texts[s] = texts[s] + [x for x in tokens[s].tolist() if x >= 0]
            counts.add(int(accepted[s]))
    assert len(counts) > 2
