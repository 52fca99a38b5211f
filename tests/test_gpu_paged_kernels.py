"""GPU: attention over a paged cache in each of its kernels: many sequences (workgroups of 4 waves) with every number of 16-row tiles,
sequences that are not split, non-finite values in several tiles, rows that start anywhere in memory."""
import pytest

from test_gpu_paged import TYPES, check, run, setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("x,cache", TYPES)
@pytest.mark.parametrize("rep,NKV,HD,T", [(1, 2, 64, 1), (4, 2, 64, 5), (7, 2, 64, 6), (4, 2, 128, 1), (4, 2, 128, 6), (7, 2, 128, 5), (3, 2, 192, 1),
                                          (5, 2, 192, 4), (4, 2, 256, 1), (7, 2, 256, 4)])
def test_many_sequences_of_every_shape(gpu, rep, NKV, HD, T, x, cache):
    import torch
    g = torch.Generator().manual_seed(HD + T)
    lens = torch.randint(0, 90, (260,), generator=g).tolist()
    lens[7], lens[100] = 1500, 700
    a = setup(torch, T, lens, T, rep * NKV, NKV, HD, 16, x, cache)
    check(run(*a), *a)


@pytest.mark.parametrize("cache", ["float16", "float32"])
def test_unsplit_long_sequence(gpu, cache):
    """More sequences than are split: one of 9000 positions is a single workgroup's, which looks its pages up several times."""
    import torch
    lens = [1] * 4200
    lens[4111] = 9000
    a = setup(torch, 2, lens, 1, 2, 1, 64, 16, "float32", cache)
    out = run(*a)
    part = slice(4100, 4120)
    check(out[part], a[0][part], a[1][part], a[2][part], a[3])
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("x,cache", TYPES)
@pytest.mark.parametrize("HD,T,n", [(64, 13, 300), (128, 5, 300), (128, 11, 70), (192, 7, 300), (256, 9, 40), (128, 11, 5000)])
@pytest.mark.parametrize("bad", [float("nan"), float("-inf")])
def test_non_finite_values_in_several_tiles(gpu, HD, T, n, bad, x, cache):
    """As the formula with masks has it: exactly the tokens from the value's position on, in its dimension."""
    import torch
    q, pos, pages, c = setup(torch, HD, [n, 20], T, 8, 2, HD, 16, x, cache)
    clean = run(q, pos, pages, c).cpu()
    hit = torch.zeros(clean.shape, dtype=torch.bool)
    for back, dim, kv in ((1, 0, 0), (2, HD - 1, 1), (T // 2 + 1, 37, 0), (T - 1, 5, 1)):  # positions among the new tokens'
        p = n - back
        c[pages[0, p // 16], 1, kv, p % 16, dim] = bad
        hit[0, T - back:, 4 * kv:4 * kv + 4, dim] = True
    out = run(q, pos, pages, c).cpu()
    assert not torch.isfinite(out[hit]).any() and torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("x,cache", TYPES)
def test_rows_that_start_anywhere(gpu, x, cache):
    import torch
    from webpytorch_amd import core
    q, pos, pages, c = (t.cuda() for t in setup(torch, 2, [40, 500], 3, 4, 2, 64, 16, x, cache))
    want = core.paged_attention(q, pos, pages, c)
    for off in (1, 3):
        buf = torch.full((q.numel() + 8,), 9.0, dtype=q.dtype, device="cuda")
        out = torch.full((q.numel() + 8,), 9.0, dtype=q.dtype, device="cuda")
        buf[off:off + q.numel()] = q.flatten()
        core.paged_attention(buf[off:off + q.numel()].view(q.shape), pos, pages, c, out=out[off:off + q.numel()].view(q.shape))
        assert torch.equal(out[off:off + q.numel()].view(q.shape), want)
        assert (out[:off] == 9).all() and (out[off + q.numel():] == 9).all()


def test_scores_of_minus_infinity(gpu):
    """Keys that leave a token no weight give zeros, as no key does; beside others they have probability 0."""
    import torch
    q, pos, pages, c = setup(torch, 2, [40, 50], 1, 2, 1, 64, 16, "float32", "float32")
    q[:] = 1.0
    c[pages[0, :3].long(), 0, 0, :, 3] = float("-inf")
    c[pages[1, 0], 0, 0, 5, 3] = float("-inf")
    out = run(q, pos, pages, c)
    assert (out[0] == 0).all()
    c[pages[0, :3].long(), 0, 0, :, 3] = -1e30  # the same probabilities: 0 beside any other key
    c[pages[1, 0], 0, 0, 5, 3] = -1e30
    check(out[1:], q[1:], pos[1:], pages[1:], c)


@pytest.mark.parametrize("S", [1, 3, 40])
def test_lengths_across_the_rule_of_parts(gpu, S):
    """Lengths around every border of steps and parts, one token of each."""
    import torch
    for n in (767, 768, 769, 1023, 1025, 2047, 2049, 4096):
        a = setup(torch, n, [n] + [max(1, n // (s + 2)) for s in range(S - 1)], 1, 2, 1, 64, 16, "float32", "float16")
        check(run(*a), *a)
