"""GPU: verification at temperatures far from 1, against float64 (`oracle/paged.py`): down to fp32's least number, where a row is all at
its largest logits, and up to its greatest, where all tokens but the masked ones are alike."""
import numpy as np
import pytest

from oracle import paged

pytestmark = pytest.mark.gpu

BORDER = 1e-11  # as tests/test_gpu_verify.py: a draw this near to a border may fall on either side


def check(x, ids, u, d, temperature):
    import torch
    from webpytorch_amd import core
    dev = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    got = core.verify_drafts(dev(x), dev(ids), dev(u), dev(d), temperature=dev(temperature) if isinstance(temperature, np.ndarray) else temperature)
    tokens, accepted, near = paged.verify(x, ids, u, d, temperature)
    assert near.min() > BORDER
    np.testing.assert_array_equal(got.accepted.cpu().numpy(), accepted)
    np.testing.assert_array_equal(got.tokens.cpu().numpy(), tokens)
    return tokens, accepted


def peaked(seed, S, D, V, top, dt):
    """Rows whose largest logit is `top`, with neighbours a step of dt or two below it, and some equal to it; the draft's without."""
    g = np.random.default_rng(seed)
    x = (g.standard_normal((S, D + 1, V)) * 3).astype(dt)
    x = np.minimum(x, dt(top) - dt(1)).astype(dt)
    d = np.minimum(x[:, :D] + (g.standard_normal((S, D, V)) * 0.5).astype(dt), dt(top) - dt(1)).astype(dt)
    step = np.nextafter(dt(top), dt(0))
    for s in range(S):
        for i in range(D + 1):
            at = g.permutation(V)[:4]
            x[s, i, at[0]] = dt(top)
            x[s, i, at[1]] = step
            x[s, i, at[2]] = dt(top) if s % 3 == 0 else np.nextafter(step, dt(0))
            if i < D:
                d[s, i, at[s % 4]] = dt(top)
    ids = np.argmax(x[:, :D], -1).astype(np.int32)
    ids[1::4] = np.argmax(d[1::4], -1)
    ids[2::5, D // 2:] = 7  # all but never a likely one
    return x, d, ids, np.maximum(g.random((S, D + 1)), 2.0 ** -20).astype(np.float32)


@pytest.mark.parametrize("dt", [np.float32, np.float16])
@pytest.mark.parametrize("top", [20.0, 150.0, -20.0, 500.0])
@pytest.mark.parametrize("t", [1e-3, 1e-6, 1e-8, 5e-9, 2e-9, 1e-10, 1e-20, 1e-38, 2e-45])
def test_small_temperatures(gpu, t, top, dt):
    t = float(np.float32(t))
    for V in (200, 9001):
        x, d, ids, u = peaked(int(abs(top)) + V, 12, 3, V, top, dt)
        tokens, accepted = check(x, ids, u, d, t)
        assert (tokens[np.arange(12), accepted] >= 0).all()
        check(x, ids, u, None, t)
        check(x[:, :1], ids[:, :0], u[:, :1], None, t)
        each = np.full(12, t, np.float32)
        each[::4] = 0.7
        check(x, ids, u, d, each)
        check(x, ids, u, None, each)


@pytest.mark.parametrize("dt", [np.float32, np.float16])
@pytest.mark.parametrize("t", [1e3, 1e30, 1e36, 1e38, 3e38])
def test_large_temperatures(gpu, t, dt):
    """All tokens are nearly alike; those masked by -inf have no weight in the rows' sums either."""
    t = float(np.float32(t))
    g = np.random.default_rng(3)
    for V in (8, 40):
        x = (g.standard_normal((96, 3, V)) * 5).astype(dt)
        x[:, :, V // 4:] = -np.inf
        x[1, :, 0] = 6e4
        d = x[:, :2] + dt(1)
        d[:, :, V // 8] = -np.inf  # the draft lacks a token
        ids = g.integers(0, V // 4, (96, 2)).astype(np.int32)
        ids[::6, 1] = V - 1        # a masked one
        u = g.random((96, 3)).astype(np.float32)
        _, accepted = check(x, ids, u, None, t)
        assert accepted.max() > 0 and accepted.min() == 0
        check(x, ids, u, d, t)
        each = np.full(96, t, np.float32)
        each[::3] = 1.0
        check(x, ids, u, d, each)
