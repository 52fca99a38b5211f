"""The 4-bit cache's rule (CPU): its error bound, its special groups, and the layout's places."""
import numpy as np
import pytest

from oracle import kv4


def test_every_value_is_within_half_a_step():
    """Half a step (S / 16), the rounding of S and Z (2^-11 of each: a code can be off by what they move the
    grid) and of the value itself."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((400, 128)) * 10.0 ** rng.uniform(-3, 3, (400, 1)) + rng.standard_normal((400, 1)) * 5).astype(np.float32)
    c, S, Z = kv4.quantize(x)
    err = np.abs(kv4.stands_for(c, S, Z) - x).reshape(400, 4, 32).max(-1)
    S, Z = S.astype(np.float64), np.abs(Z.astype(np.float64))
    assert (err <= S / 32 + 2.0 ** -11 * (2 * S + Z) + 2.0 ** -11 * (2 * S + Z) + 2.0 ** -24).all()


@pytest.mark.parametrize("v", [0.0, 1.0, -3.25, 1e-9, 6e-8, -2e-7, 16384.0, -1e30, 1e30])
def test_constant_groups(v):
    c, S, Z = kv4.quantize(np.full((1, 32), v, np.float32))
    got = kv4.stands_for(c, S, Z)
    want = float(np.clip(v, -16384, 16384))
    assert np.isfinite(got).all() and np.abs(got - want).max() <= 2.0 ** -11 * abs(want) + 2.0 ** -25


def test_non_finite_groups_read_as_nan():
    x = np.ones((3, 64), np.float32)
    x[0, 3], x[1, 40] = np.nan, np.inf
    got = kv4.stands_for(*kv4.quantize(x))
    assert np.isnan(got[0, :32]).all() and np.isnan(got[1, 32:]).all()
    assert np.isfinite(got[0, 32:]).all() and np.isfinite(got[1, :32]).all() and np.isfinite(got[2]).all()


@pytest.mark.parametrize("HD", [64, 128, 192, 256])
def test_places_cover_the_record_once(HD):
    (kw, kb), (vw, vb), km, vm = kv4._places(HD)
    bits = np.concatenate([(w * 8 + b)[..., None] + np.arange(4) for w, b in ((kw, kb), (vw, vb))]).ravel()
    halves = np.concatenate([(m * 8)[..., None] + np.arange(16) for m in km + vm]).ravel()
    assert np.array_equal(np.sort(np.concatenate([bits, halves])), np.arange(40 * HD * 8))
