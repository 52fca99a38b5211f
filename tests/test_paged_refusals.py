"""Refusals of the rotation, the paged cache's operators and the verification (CPU): what they do not cover raises before
anything is launched."""
import ctypes

import numpy as np
import pytest

from webpytorch_amd import _lib

P = 1 << 20  # addresses that no refused call reads, far apart
Q, R = 1 << 40, 1 << 41


def call(name, **over):
    d = {
        "miq_rope": dict(x=P, dt=0, ld=128, lh=64, pos=P, cos=P, sin=P, rows=8, rot=64, pairs=0, transpose=0, out=Q, old=128, olh=64, T=3, H=2,
                         HD=64, stream=None),
        "miq_paged_append": dict(qkv=P, dt=0, ld=256, qn=None, kn=None, eps=1e-6, pos=P, pages=P, most=2, cos=P, sin=P, rows=8, rot=64, pairs=0,
                                 q=Q, cache=R, cdt=1, num=4, page=16, S=1, T=1, NH=2, NKV=1, HD=64, stream=None),
        "miq_paged_attention": dict(q=P, dt=0, cache=R, cdt=1, num=4, page=16, pos=P, pages=P, most=2, out=Q, S=1, T=1, NH=2, NKV=1, HD=64,
                                    scale=1.0, ws=None, wsb=0, stream=None),
        "miq_verify_drafts": dict(x=P, dt=0, ls=3000, lr=1000, ids=P, d=None, ds=2000, dr=1000, u=P, temps=None, temp=1.0, tokens=Q, acc=Q, S=2, D=2,
                                  V=1000, ws=R, wsb=1 << 30, stream=None),
    }[name]
    assert set(over) <= set(d)
    d.update(over)
    return _lib.call(name, *d.values())


@pytest.mark.parametrize("name,over,exc,text", [
    ("miq_rope", dict(HD=63), ValueError, "HD=63"),
    ("miq_rope", dict(HD=2048), ValueError, "HD=2048"),
    ("miq_rope", dict(rot=66), ValueError, "rot=66"),
    ("miq_rope", dict(rot=0), ValueError, "rot=0"),
    ("miq_rope", dict(rot=31), ValueError, "rot=31"),
    ("miq_rope", dict(rows=0), ValueError, "rows=0"),
    ("miq_rope", dict(T=-1), ValueError, "T=-1"),
    ("miq_rope", dict(dt=2), NotImplementedError, "dtype 2"),
    ("miq_rope", dict(ld=127), ValueError, "overlap"),
    ("miq_rope", dict(lh=63), ValueError, "overlap"),
    ("miq_rope", dict(old=100), ValueError, "overlap"),
    ("miq_rope", dict(olh=-64), ValueError, "overlap"),
    ("miq_rope", dict(ld=1 << 50), ValueError, "overlap"),
    ("miq_rope", dict(out=None), ValueError, "null"),
    ("miq_rope", dict(cos=None), ValueError, "null"),
    ("miq_rope", dict(out=P + 16), ValueError, "apart"),
    ("miq_rope", dict(out=P, old=256), ValueError, "apart"),
    ("miq_rope", dict(out=P - 1400), ValueError, "apart"),
    ("miq_rope", dict(T=(1 << 31) - 1, out=1 << 60), NotImplementedError, "past the grid"),
    ("miq_paged_append", dict(HD=80, ld=4096), NotImplementedError, "HD=80"),
    ("miq_paged_append", dict(page=8), NotImplementedError, "8 positions"),
    ("miq_paged_append", dict(page=48), NotImplementedError, "48 positions"),
    ("miq_paged_append", dict(page=8192), NotImplementedError, "8192 positions"),
    ("miq_paged_append", dict(most=1 << 27), NotImplementedError, "2.30 positions"),
    ("miq_paged_append", dict(num=0), ValueError, "of 0"),
    ("miq_paged_append", dict(ld=255), ValueError, "255"),
    ("miq_paged_append", dict(rot=65), ValueError, "rot=65"),
    ("miq_paged_append", dict(rows=0), ValueError, "rows=0"),
    ("miq_paged_append", dict(cdt=2), NotImplementedError, "dtypes 0, 2"),
    ("miq_paged_append", dict(cache=R + 8), ValueError, "aligned"),
    ("miq_paged_append", dict(q=None), ValueError, "null"),
    ("miq_paged_append", dict(pages=None), ValueError, "null"),
    ("miq_paged_append", dict(cos=None), ValueError, "null"),
    ("miq_paged_append", dict(q=P + 512), ValueError, "apart"),
    ("miq_paged_append", dict(qkv=R + 1024), ValueError, "apart"),
    ("miq_paged_append", dict(q=R - 64), ValueError, "apart"),
    ("miq_paged_append", dict(S=1 << 20, T=1 << 12), NotImplementedError, "past the grid"),
    ("miq_paged_attention", dict(HD=96), NotImplementedError, "HD=96"),
    ("miq_paged_attention", dict(NH=3, NKV=2), ValueError, "NKV=2"),
    ("miq_paged_attention", dict(NKV=0), ValueError, "NKV=0"),
    ("miq_paged_attention", dict(page=24), NotImplementedError, "24 positions"),
    ("miq_paged_attention", dict(dt=3), NotImplementedError, "dtypes 3"),
    ("miq_paged_attention", dict(most=4096), ValueError, "workspace"),
    ("miq_paged_attention", dict(most=4096, ws=R + 8, wsb=1 << 30), ValueError, "aligned"),
    ("miq_paged_attention", dict(scale=float("inf")), ValueError, "scale"),
    ("miq_paged_attention", dict(scale=float("nan")), ValueError, "scale"),
    ("miq_paged_attention", dict(out=None), ValueError, "null"),
    ("miq_paged_attention", dict(pos=None), ValueError, "null"),
    ("miq_paged_attention", dict(out=P), ValueError, "apart"),
    ("miq_paged_attention", dict(out=R + 4096), ValueError, "apart"),
    ("miq_paged_attention", dict(cache=R + 4), ValueError, "aligned"),
    ("miq_paged_attention", dict(S=1 << 23), NotImplementedError, "past the grid"),
    ("miq_verify_drafts", dict(D=33), NotImplementedError, "D=33"),
    ("miq_verify_drafts", dict(D=-1), ValueError, "D=-1"),
    ("miq_verify_drafts", dict(V=0), ValueError, "V=0"),
    ("miq_verify_drafts", dict(S=20000), NotImplementedError, "S=20000"),
    ("miq_verify_drafts", dict(dt=2), NotImplementedError, "dtype 2"),
    ("miq_verify_drafts", dict(lr=999), ValueError, "999"),
    ("miq_verify_drafts", dict(ls=-1), ValueError, "apart"),
    ("miq_verify_drafts", dict(d=P, dr=999), ValueError, "999"),
    ("miq_verify_drafts", dict(temp=-0.5), ValueError, "temperature"),
    ("miq_verify_drafts", dict(temp=float("nan")), ValueError, "temperature"),
    ("miq_verify_drafts", dict(temp=float("inf")), ValueError, "temperature"),
    ("miq_verify_drafts", dict(x=P + 2), ValueError, "aligned"),
    ("miq_verify_drafts", dict(u=None), ValueError, "null"),
    ("miq_verify_drafts", dict(ids=None), ValueError, "null"),
    ("miq_verify_drafts", dict(wsb=1 << 20), ValueError, "workspace"),
    ("miq_verify_drafts", dict(ws=None), ValueError, "workspace"),
    ("miq_verify_drafts", dict(ws=R + 16), ValueError, "aligned")])
def test_entry_points_refuse(name, over, exc, text):
    with pytest.raises(exc, match=text):
        call(name, **over)


def test_nothing_to_do_is_no_error():
    assert call("miq_rope", T=0) == 0 and call("miq_rope", H=0) == 0
    for name in ("miq_paged_append", "miq_paged_attention"):
        assert call(name, S=0) == 0 and call(name, T=0) == 0
    assert call("miq_verify_drafts", S=0) == 0


def test_workspaces():
    n = ctypes.c_size_t(0)
    _lib.call("miq_paged_attention_workspace", 1, 1, 4, 1, 64, 16, 4, 1, ctypes.byref(n))
    assert n.value == 0  # 64 positions: one part
    _lib.call("miq_paged_attention_workspace", 1, 1, 4, 1, 64, 16, 4096, 1, ctypes.byref(n))
    assert n.value > 4 << 20
    _lib.call("miq_verify_drafts_workspace", 0, 4, 1000, ctypes.byref(n))
    assert n.value == 0
    with pytest.raises(NotImplementedError, match="D=40"):
        _lib.call("miq_verify_drafts_workspace", 1, 40, 1000, ctypes.byref(n))


def test_tensors_off_the_gpu_are_refused():
    import torch
    from webpytorch_amd import core
    z, i32 = torch.zeros, torch.int32
    with pytest.raises(ValueError, match="on the GPU"):
        core.rope(z(1, 2, 64), z(1, dtype=i32), core.Rope(z(8, 32), z(8, 32), False))
    with pytest.raises(ValueError, match="on the GPU"):
        core.paged_append(z(1, 1, 256), z(1, 1, dtype=i32), z(1, 1, dtype=i32), z(2, 2, 1, 16, 64), 2)
    with pytest.raises(ValueError, match="on the GPU"):
        core.paged_attention(z(1, 1, 2, 64), z(1, 1, dtype=i32), z(1, 1, dtype=i32), z(2, 2, 1, 16, 64))
    with pytest.raises(ValueError, match="on the GPU"):
        core.verify_drafts(z(1, 2, 8), z(1, 1, dtype=i32), z(1, 2))


def test_caches_and_tables_that_are_refused():
    import torch
    from webpytorch_amd import core
    with pytest.raises(NotImplementedError, match="not 80"):
        core.paged_cache(4, 1, 16, 80)
    for page in (8, 24, 8192):
        with pytest.raises(ValueError, match="page="):
            core.paged_cache(4, 1, page, 64)
    with pytest.raises(TypeError, match="bfloat16"):
        core.paged_cache(4, 1, 16, 64, torch.bfloat16)
    for args, exc, text in (((0, 64), ValueError, "n=0"), ((8, 63), ValueError, "rot=63"),
                            ((8, 64, 1e4, {"rope_type": "spiral"}), NotImplementedError, "spiral"),
                            ((8, 64, 1e4, {"rope_type": "yarn", "factor": 2.0}), ValueError, "original"),
                            ((8, 64, 1e4, {"rope_type": "linear", "factor": 0.0}), ValueError, "factor=0"),
                            ((8, 64, -1.0), ValueError, "theta"),
                            ((8, 64, 1e4, {"rope_type": "wavelength", "factor": 2.0, "original_max_position_embeddings": 64, "low_freq_factor": 4.0}),
                             ValueError, "low_freq")):
        with pytest.raises(exc, match=text):
            core.rope_tables(*args)


def test_the_verdict_of_the_oracle_by_hand():
    """p = (1/2, 1/4, 1/4), q = (1/4, 1/2, 1/4): draft 1 is accepted below u = 1/2, else the token is 0."""
    from oracle import paged
    p, q = np.log([[[0.5, 0.25, 0.25], [0.25, 0.25, 0.5]]]), np.log([[[0.25, 0.5, 0.25]]])
    for u, want, n in (([0.49, 0.1], [1, 0], 1), ([0.49, 0.3], [1, 1], 1), ([0.49, 0.9], [1, 2], 1), ([0.51, 0.9], [0, -1], 0)):
        tokens, accepted, _ = paged.verify(p, np.array([[1]], np.int32), np.array([u], np.float32), q)
        assert tokens.tolist() == [want] and accepted.tolist() == [n]
    tokens, accepted, _ = paged.verify(p, np.array([[1]], np.int32), np.array([[0.3, 0.9]], np.float32))  # looked up: u < 1/4
    assert tokens.tolist() == [[2, -1]] and accepted.tolist() == [0]
