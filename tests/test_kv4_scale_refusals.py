"""Scales of the 4-bit cache's attention that are no finite number (CPU): refused, where a NaN would weigh all keys alike."""
import math

import pytest

from webpytorch_amd import _lib


@pytest.mark.parametrize("dt", [0, 1])
@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 3e38])
def test_scales(dt, scale):
    with pytest.raises(ValueError, match="scale="):
        _lib.call("miq_attention_kv4", 1 << 20, dt, 1 << 24, 256, 1 << 22, 1, 2, 1, 64, 64, scale, None, 0, None)
