"""Scalings that `core.rope_tables` does not know (CPU): a key that would change the tables is refused, not passed over."""
import numpy as np
import pytest

from webpytorch_amd import core

YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}
WAVES = {"rope_type": "llama3", "factor": 8.0, "original_max_position_embeddings": 64}


@pytest.fixture
def on_host(monkeypatch):
    monkeypatch.setattr(core, "to_device", lambda a, *_: a)


@pytest.mark.parametrize("scaling,key", [
    (dict(YARN, mscale=1.0, mscale_all_dim=1.0), "mscale"), (dict(YARN, mscale_all_dim=0.7), "mscale_all_dim"), (dict(YARN, truncate=False), "truncate"),
    (dict(YARN, low_freq_factor=1.0), "low_freq_factor"), (dict(WAVES, beta_fast=32.0), "beta_fast"), (dict(WAVES, attention_factor=1.2), "attention_factor"),
    ({"type": "linear", "factor": 2.0, "attention_factor": 1.2}, "attention_factor"), ({"type": "linear", "factor": 2.0, "short_factor": [1.0]}, "short_factor"),
    ({"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 4, "alpha": 8.0}, "alpha"), ({"factor": 4.0}, "factor"),
    ({"rope_type": "default", "factor": 4.0}, "factor"), (dict(YARN, partial_rotary_factor=0.5), "partial_rotary_factor")])
def test_unknown_keys(on_host, scaling, key):
    with pytest.raises(NotImplementedError, match=key):
        core.rope_tables(16, 64, 1e4, scaling)


@pytest.mark.parametrize("scaling,text", [
    ({"rope_type": "linear"}, "factor"), (dict(YARN, factor=None), "factor"), ({"rope_type": "dynamic", "original_max_position_embeddings": 4}, "factor"),
    ({"rope_type": "wavelength", "original_max_position_embeddings": 4}, "factor"), ({"rope_type": "linear", "factor": float("inf")}, "factor=inf"),
    (dict(YARN, rope_theta=1e6), "rope_theta")])
def test_what_a_scaling_needs(on_host, scaling, text):
    with pytest.raises(ValueError, match=text):
        core.rope_tables(16, 64, 1e4, scaling)


@pytest.mark.parametrize("base", [YARN, WAVES, {"rope_type": "linear", "factor": 2.0}, {"rope_type": "default"}])
def test_keys_that_change_nothing(on_host, base):
    """The base's own angle, a length that linear scaling has no use for, and keys that are there without a value."""
    want = core.rope_tables(16, 64, 1e4, base)
    extra = dict(base, rope_theta=1e4, original_max_position_embeddings=64, mscale=None, attention_factor=None, beta_fast=None)
    if base is YARN:
        extra["truncate"] = True
    got = core.rope_tables(16, 64, 1e4, extra)
    np.testing.assert_array_equal(got.cos, want.cos)
    np.testing.assert_array_equal(got.sin, want.sin)
