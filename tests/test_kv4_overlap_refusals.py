"""Overlapping inputs and outputs of the decoder operators (CPU): refused by their addresses, before anything is launched."""
import pytest

from webpytorch_amd import _lib

QKV, W = 1 << 20, 256 * 4  # two query heads and one of k and v, of 64 fp32 values: T rows of 1024 bytes
CACHE = 64 * 64 * 4        # bytes of an fp32 cache of 64 positions; the 4-bit one has 2 x 2560


def rope(T=1, ld=256, q=1 << 24, kc=1 << 25, vc=1 << 26, four=False):
    if four:
        return _lib.call("miq_qk_norm_rope_kv4", QKV, 0, ld, None, None, 1e-6, 256, 256, 256, q, kc, T, 2, 1, 64, 64, None)
    return _lib.call("miq_qk_norm_rope_kv", QKV, ld, None, None, 1e-6, 256, 256, 256, q, kc, vc, T, 2, 1, 64, 64, None)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("kw", [dict(q=QKV), dict(q=QKV + W - 4), dict(q=QKV - 2 * 64 * 4 + 4), dict(q=QKV + 256),
                                dict(T=3, q=QKV + 3 * W - 4), dict(T=3, ld=1024, q=QKV + 2 * 4096), dict(T=3, ld=1024, q=QKV + 2 * 4096 + W - 4),
                                dict(T=3, ld=512, q=QKV + W), dict(T=3, ld=1024, q=QKV - 3 * 512 + 4)])
def test_queries_and_rows(kw, four):
    with pytest.raises(ValueError, match="apart from qkv"):
        rope(four=four, **kw)


@pytest.mark.parametrize("kw", [dict(kc=QKV), dict(kc=QKV - 16), dict(kc=QKV + W - 16), dict(kc=1 << 24), dict(kc=(1 << 24) + 496)])
def test_cache_with_rows_and_queries(kw):
    for four in (False, True):
        with pytest.raises(ValueError, match="cache must lie apart"):
            rope(four=four, **kw)
    with pytest.raises(ValueError, match="cache must lie apart"):
        rope(vc=kw["kc"])


@pytest.mark.parametrize("off", [0, 4, CACHE - 4, 4 - CACHE])
def test_two_caches(off):
    with pytest.raises(ValueError, match="caches overlap"):
        rope(vc=(1 << 25) + off)


@pytest.mark.parametrize("dt", [0, 1])
@pytest.mark.parametrize("off", [0, 2, -2, 254, -254])
def test_attention(dt, off):
    q, cache, n = 1 << 20, 1 << 24, 3 * 2 * 64 * (4 if dt == 0 else 2)
    run = lambda out: _lib.call("miq_attention_kv4", q, dt, cache, 256, out, 3, 2, 1, 64, 64, 1.0, None, 0, None)  # noqa: E731
    with pytest.raises(ValueError, match="apart from q"):
        run(q + off)
    with pytest.raises(ValueError, match="apart from q"):
        run(q + (n - 2 if off >= 0 else 2 - n))
    with pytest.raises(ValueError, match="apart from the cache"):
        run(cache + 16 * abs(off))  # of 5120 bytes
    with pytest.raises(ValueError, match="apart from the cache"):
        run(cache - n + 2)
