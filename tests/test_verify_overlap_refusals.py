"""Answers of the verification over what it still reads, or over each other (CPU): refused by their addresses, before anything is launched."""
import pytest

from webpytorch_amd import _lib


def verify(**over):
    # 3 sequences of 2 drafts, V = 100, rows and sequences one after the other
    d = dict(x=1 << 24, dt=0, ls=300, lr=100, ids=1 << 25, d=1 << 26, ds=200, dr=100, u=1 << 27, temps=1 << 28, temp=1.0, tokens=1 << 29, acc=1 << 30,
             S=3, D=2, V=100, ws=1 << 31, wsb=1 << 30, stream=None)
    d.update(over)
    return _lib.call("miq_verify_drafts", *d.values())


@pytest.mark.parametrize("name,n", [("tokens", 36), ("acc", 12)])
@pytest.mark.parametrize("at,size", [(1 << 24, 3600), (1 << 25, 24), (1 << 26, 2400), (1 << 27, 36), (1 << 28, 12)])
def test_answers_over_inputs(name, n, at, size):
    for off in (0, size - 4, 4 - n):
        with pytest.raises(ValueError, match="apart"):
            verify(**{name: at + off})


@pytest.mark.parametrize("over", [dict(tokens=1 << 30), dict(acc=(1 << 29) + 32), dict(tokens=1 << 31), dict(acc=(1 << 31) + (1 << 20)),
                                  dict(x=(1 << 29) - 3600 + 4), dict(dt=1, x=(1 << 29) - 1800 + 2), dict(S=1, ls=1 << 60, tokens=(1 << 24) + 1196)])
def test_answers_over_each_other_or_the_workspace(over):
    with pytest.raises(ValueError, match="apart"):
        verify(**over)


def test_sequences_too_far_apart():
    for over in (dict(ls=1 << 60), dict(ds=1 << 60)):
        with pytest.raises(ValueError, match="apart"):
            verify(**over)
