"""Outputs of the rotation over what it still reads (CPU): refused by their addresses, before anything is launched."""
import pytest

from webpytorch_amd import _lib

X, POS, COS, SIN, OUT = (1 << n for n in (24, 26, 28, 30, 32))  # x and out: 3 tokens of 2 heads of 64 fp32 values, tables of 8 rows


def rope(out, x=X, T=3):
    return _lib.call("miq_rope", x, 0, 128, 64, POS, COS, SIN, 8, 64, 0, 0, out, 128, 64, T, 2, 64, None)


@pytest.mark.parametrize("out", [POS, POS + 8, POS - 3 * 512 + 4, COS, COS + 8 * 32 * 4 - 4, SIN, SIN - 3 * 512 + 4, SIN + 1020])
def test_a_rotation_over_its_positions_or_tables(out):
    with pytest.raises(ValueError, match="apart"):
        rope(out)


def test_a_rotation_in_place_over_its_positions():
    with pytest.raises(ValueError, match="apart"):
        rope(POS, x=POS)
