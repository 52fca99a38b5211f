"""GPU: a temperature given as a number is the law's own, not the fp32 number next to it. 0.6 and 0.8 lie 1.5e-8 to 4e-8 (relative) from fp32's: with
random numbers between a border of the one law and of the other, a draw tells them apart."""
import numpy as np
import pytest

from oracle import paged
from test_gpu_verify_temperatures import check, peaked

pytestmark = pytest.mark.gpu

# The kernel's probabilities are off by 3e-13 (tests/test_gpu_verify.py). A border between tokens moves by up to 1e-8 with fp32's temperature.
BORDER = 1e-11


def row_of(seed, V, peak, dt):
    g = np.random.default_rng(seed)
    return (g.standard_normal(V) * peak).astype(dt)


def last_below(b):
    """The largest fp32 numbers that are not above b."""
    f = b.astype(np.float32)
    return np.where(f.astype(np.float64) > b, np.nextafter(f, np.float32(0)), f).astype(np.float32)


def between(row, t, n):
    """n fp32 numbers u, each behind a border of the law at one of t and float32(t) and ahead of it at the other."""
    runs = [np.cumsum(paged.law(row, x)) for x in (t, float(np.float32(t)))]
    runs = [r / r[-1] for r in runs]
    u = np.unique(last_below(np.maximum(*runs)))
    u = u[(u > 2.0 ** -10) & (u < 1)]
    tokens = [np.searchsorted(r, u.astype(np.float64), side="right") for r in runs]
    at = np.clip(tokens[0], 1, len(row) - 1)
    far = np.minimum(np.abs(runs[0][at] - u), np.abs(runs[0][at - 1] - u)) > BORDER
    u = u[(tokens[0] != tokens[1]) & far]
    return u[np.linspace(0, len(u) - 1, n).astype(int)]


@pytest.mark.parametrize("dt", [np.float32, np.float16])
@pytest.mark.parametrize("V,t", [(151936, 0.6), (128256, 0.8), (32003, 0.7)])
def test_draws_near_borders(gpu, V, t, dt):
    import torch
    from webpytorch_amd import core
    S = 48
    for seed, peak in ((1, 1.5), (2, 3.0)):
        row = row_of(seed, V, peak, dt)
        u = between(row, t, S)[:, None]
        x = np.broadcast_to(row, (S, 1, V))
        want, _, near = paged.verify(x, np.zeros((S, 0), np.int32), u, None, t)
        other, _, _ = paged.verify(x, np.zeros((S, 0), np.int32), u, None, float(np.float32(t)))
        assert near.min() > BORDER and (want != other).sum() > S // 2
        got = core.verify_drafts(torch.from_numpy(row).cuda().expand(S, 1, V), torch.zeros((S, 0), dtype=torch.int32, device="cuda"),
                                 torch.from_numpy(u).cuda(), temperature=t)
        np.testing.assert_array_equal(got.tokens.cpu().numpy(), want)
        # and a temperature of each sequence is that fp32 number
        got = core.verify_drafts(torch.from_numpy(row).cuda().expand(S, 1, V), torch.zeros((S, 0), dtype=torch.int32, device="cuda"),
                                 torch.from_numpy(u).cuda(), temperature=torch.full((S,), t, device="cuda"))
        sure = paged.verify(x, np.zeros((S, 0), np.int32), u, None, float(np.float32(t)))[2] > BORDER
        np.testing.assert_array_equal(got.tokens.cpu().numpy()[sure], other[sure])


@pytest.mark.parametrize("t", [0.6, 0.8, 0.7])
def test_acceptance_near_its_border(gpu, t):
    """Looked-up drafts with u between p at t and p at float32(t): accepted by the one and not by the other."""
    import torch
    from webpytorch_amd import core
    V, S = 20000, 64
    row = row_of(5, V, 2.0, np.float32)
    p, q = paged.law(row, t), paged.law(row, float(np.float32(t)))
    u = last_below(np.maximum(p, q))
    ids = np.flatnonzero(((u < p) != (u < q)) & (np.abs(u / p - 1) > 1e-11) & (np.abs(u / q - 1) > 1e-11))[:S]
    assert len(ids) == S
    x = np.broadcast_to(row, (S, 2, V))
    u = np.stack([u[ids], np.full(S, 0.5, np.float32)], 1)
    tokens, accepted, near = paged.verify(x, ids[:, None].astype(np.int32), u, None, t)
    assert near.min() > BORDER and (accepted == (p[ids] > q[ids])).all()
    got = core.verify_drafts(torch.from_numpy(row).cuda().expand(S, 2, V), torch.from_numpy(ids[:, None].astype(np.int32)).cuda(),
                             torch.from_numpy(u).cuda(), temperature=t)
    np.testing.assert_array_equal(got.accepted.cpu().numpy(), accepted)
    np.testing.assert_array_equal(got.tokens.cpu().numpy(), tokens)


@pytest.mark.parametrize("t", [1e-50, 1e-300, 5e-324, 1e39, 1e200])
@pytest.mark.filterwarnings("ignore:overflow encountered")
def test_numbers_past_fp32(gpu, t):
    """All at the largest logits, or all tokens but the masked ones alike."""
    x, d, ids, u = peaked(11, 12, 3, 900, 20.0, np.float32)
    x[:, :, 300:500] = -np.inf
    x[:, :, 250] = 20.0
    ids[3::4] = 270
    check(x, ids, u, d, t)
    check(x, ids, u, None, t)
    check(x[:, :1], ids[:, :0], u[:, :1], None, t)
