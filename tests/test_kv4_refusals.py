"""Refusals of the decoder operators (CPU): what they do not cover raises before anything is launched."""
import ctypes

import pytest

from webpytorch_amd import _lib

P = 256  # a non-null address that no refused call reads


def call(name, **over):
    d = {
        "miq_qk_norm_rope_kv": dict(qkv=P, ld=256, qn=None, kn=None, eps=1e-6, state=P, cos=P, sin=P, q=P, kc=P, vc=P, T=1, NH=2,
                                    NKV=1, HD=64, LMAX=8, stream=None),
        "miq_qk_norm_rope_kv4": dict(qkv=P, dt=0, ld=256, qn=None, kn=None, eps=1e-6, state=P, cos=P, sin=P, q=P, cache=P, T=1, NH=2,
                                     NKV=1, HD=64, LMAX=8, stream=None),
        "miq_kv4_dequant_f32": dict(cache=P, k=P, v=P, NKV=1, LMAX=64, HD=64, start=0, n=4, stream=None),
        "miq_attention_kv4": dict(q=P, dt=0, cache=P, state=P, out=P, T=1, NH=2, NKV=1, HD=64, LMAX=8, scale=1.0, ws=None, wsb=0,
                                  stream=None),
        "miq_token_logprobs": dict(x=P, dt=0, ld=1000, ids=P, T=1, V=1000, k=0, lp=P, ent=P, rank=P, ti=P, tl=P, state=None, rows=1,
                                   ws=None, wsb=0, stream=None),
    }[name]
    d.update(over)
    return _lib.call(name, *d.values())


@pytest.mark.parametrize("name,over,exc,text", [
    ("miq_qk_norm_rope_kv", dict(NH=3, NKV=2), ValueError, "NKV=2"),
    ("miq_qk_norm_rope_kv", dict(HD=63), ValueError, "HD=63"),
    ("miq_qk_norm_rope_kv", dict(HD=288, ld=4096), ValueError, "HD=288"),
    ("miq_qk_norm_rope_kv", dict(ld=255), ValueError, "255 values|rows 255"),
    ("miq_qk_norm_rope_kv", dict(kc=None), ValueError, "null"),
    ("miq_qk_norm_rope_kv", dict(T=-1), ValueError, "T=-1"),
    ("miq_qk_norm_rope_kv", dict(T=1 << 26), NotImplementedError, "past the grid"),
    ("miq_qk_norm_rope_kv4", dict(T=1 << 26), NotImplementedError, "past the grid"),
    ("miq_qk_norm_rope_kv4", dict(HD=80, ld=4096), NotImplementedError, "HD=80"),
    ("miq_qk_norm_rope_kv4", dict(dt=2), NotImplementedError, "dtype 2"),
    ("miq_qk_norm_rope_kv4", dict(cache=264), ValueError, "aligned"),
    ("miq_qk_norm_rope_kv4", dict(state=None), ValueError, "null"),
    ("miq_kv4_dequant_f32", dict(start=60, n=5), ValueError, "start=60"),
    ("miq_kv4_dequant_f32", dict(HD=96), NotImplementedError, "HD=96"),
    ("miq_attention_kv4", dict(HD=32), NotImplementedError, "HD=32"),
    ("miq_attention_kv4", dict(NH=3, NKV=2), ValueError, "NKV=2"),
    ("miq_attention_kv4", dict(LMAX=1 << 20), ValueError, "workspace"),
    ("miq_attention_kv4", dict(q=None), ValueError, "null"),
    ("miq_attention_kv4", dict(dt=1, out=None), ValueError, "null"),
    ("miq_attention_kv4", dict(cache=260), ValueError, "aligned"),
    ("miq_attention_kv4", dict(LMAX=0), ValueError, "LMAX=0"),
    ("miq_token_logprobs", dict(k=33), NotImplementedError, "k=33"),
    ("miq_token_logprobs", dict(k=5, V=4), ValueError, "k=5"),
    ("miq_token_logprobs", dict(ld=999), ValueError, "999"),
    ("miq_token_logprobs", dict(V=151936, ld=151936), ValueError, "workspace"),
    ("miq_token_logprobs", dict(T=65536), NotImplementedError, "65536"),
    ("miq_token_logprobs", dict(T=2, state=P), ValueError, "one row"),
    ("miq_token_logprobs", dict(x=258), ValueError, "aligned"),
    ("miq_token_logprobs", dict(ids=None), ValueError, "null")])
def test_entry_points_refuse(name, over, exc, text):
    with pytest.raises(exc, match=text):
        call(name, **over)


def test_nothing_to_do_is_no_error():
    for name in ("miq_qk_norm_rope_kv", "miq_qk_norm_rope_kv4", "miq_attention_kv4", "miq_token_logprobs"):
        assert call(name, T=0) == 0
    assert call("miq_kv4_dequant_f32", n=0) == 0


def test_cache_bytes():
    n = ctypes.c_size_t(0)
    _lib.call("miq_kv4_cache_bytes", 2, 33, 64, ctypes.byref(n))
    assert n.value == 2 * 2 * 40 * 64
    with pytest.raises(NotImplementedError):
        _lib.call("miq_kv4_cache_bytes", 2, 33, 80, ctypes.byref(n))


def test_tensors_off_the_gpu_are_refused():
    import torch
    from webpytorch_amd import core
    z = torch.zeros
    with pytest.raises(ValueError, match="on the GPU"):
        core.token_logprobs(z(2, 8), z(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="on the GPU"):
        core.attention_kv4(z(1, 2, 64), z(1, 1, 2560, dtype=torch.uint8), z(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="on the GPU"):
        core.qk_norm_rope(z(1, 256), z(1, dtype=torch.int32), z(8, 32), z(8, 32), 2, (z(1, 8, 64), z(1, 8, 64)))
    with pytest.raises(NotImplementedError, match="not 80"):
        core.kv4_cache(1, 8, 80)


def test_context_length_of_a_four_bit_cache():
    from webpytorch_amd import checkpoint
    assert checkpoint.auto_lmax(None, 10 ** 7, 24, 2, 64, 4) == (2 << 30) // (2 * 24 * 2 * 64 * 5 // 8)
    assert checkpoint.auto_lmax(None, 4096, 24, 2, 64, 4) == 4096
