"""GPU: position rotation in its layouts, and the rotation with the append to a paged cache, against float64
(`oracle/paged.py`)."""
import math

import numpy as np
import pytest

from oracle import paged

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -11  # half a step of fp32 and fp16, relative
# A rotated value is fma(x, c, -(y s)): a rounding of the product y s and one of the sum, at most 2 U32 (|x c| + |y s|) and
# terms of U32^2. With a norm: 8 squares of a thread in a chain of fmas and 5 sums of threads (13 U32 of the sum of squares, half
# of it in the root), the division by HD, the sum with eps and the root (3), the quotient (1) and two products (2): 13 U32 more.
ROTATED, NORMED = 3 * U32, 16 * U32


def angles(torch, n, rot, theta=1e4):
    a = np.arange(n, dtype=np.float64)[:, None] / (theta ** (np.arange(0, rot, 2, dtype=np.float64) / rot))
    return torch.from_numpy(np.cos(a).astype(np.float32)).cuda(), torch.from_numpy(np.sin(a).astype(np.float32)).cuda()


def near(got, want, mag, rel, half):
    """Within rel * mag, and for an fp16 result half a step of it (2^-25 in its subnormal range)."""
    got = got.double().cpu().numpy()
    assert got.shape == want.shape
    tol = rel * mag + ((U16 * (np.abs(want) + rel * mag) + 2.0 ** -25) if half else U32 * np.abs(want) + 1e-44)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol).all(), np.abs((got - want) / np.maximum(tol, 1e-60)).max()


@pytest.mark.parametrize("dt", ["float32", "float16"])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("T,H,HD,rot", [(1, 1, 64, 64), (3, 5, 128, 64), (2, 4, 80, 40), (7, 3, 96, 20), (1, 2, 2, 2), (5, 2, 10, 6),
                                        (300, 30, 128, 128), (700, 12, 192, 48), (257, 33, 64, 16), (2, 3, 1024, 1024)])
def test_rope(gpu, T, H, HD, rot, pairs, dt):
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(T * 31 + HD)
    cos, sin = angles(torch, 500, rot)
    x = (torch.randn((T, H, HD), generator=g) * 3).to(getattr(torch, dt)).cuda()
    pos = torch.randint(0, 500, (T,), generator=g, dtype=torch.int32)
    pos[0] = 499
    for transpose in (False, True):
        got = core.rope(x, pos.cuda(), core.Rope(cos, sin, pairs), transpose=transpose)
        want, mag = paged.rope(x.cpu().numpy(), pos.numpy(), cos.cpu().numpy(), sin.cpu().numpy(), pairs, transpose)
        near(got, want, mag, ROTATED, dt == "float16")
        if rot < HD:
            assert torch.equal(got[..., rot:], x[..., rot:])


@pytest.mark.parametrize("dt", ["float32", "float16"])
@pytest.mark.parametrize("pairs", [False, True])
def test_rope_of_slices_views_and_in_place(gpu, pairs, dt):
    """Rows within wider ones, odd distances, heads ahead of tokens, unaligned starts; in place, and into a slice."""
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(5)
    T, H, HD, rot = 9, 3, 64, 32
    r = core.Rope(*angles(torch, 40, rot), pairs)
    pos = torch.arange(3, 3 + T, dtype=torch.int32).cuda()
    big = torch.randn(4096, generator=g).to(getattr(torch, dt)).cuda()
    views = [big[:T * 256].view(T, 256)[:, :H * HD].unflatten(1, (H, HD)),
             big[1:1 + T * 199].view(T, 199)[:, 2:2 + H * HD].unflatten(1, (H, HD)),
             big[:T * H * 66].view(T, H, 66)[..., :HD], big[:H * T * HD].view(H, T, HD).transpose(0, 1),
             big[:T * H * HD].view(T, HD, H).transpose(1, 2)]
    for v in views:
        want = core.rope(v.clone(memory_format=torch.contiguous_format), pos, r)
        assert torch.equal(core.rope(v, pos, r), want)
        if v.stride(2) == 1:
            own = torch.zeros_like(big).as_strided(v.shape, v.stride(), v.storage_offset())
            own.copy_(v)
            core.rope(own, pos, r, out=own)
            assert torch.equal(own, want)
    rows = torch.full((T, 7 + H * HD), 5.0, dtype=big.dtype, device="cuda")
    core.rope(views[0], pos, r, out=rows[:, 4:4 + H * HD].unflatten(1, (H, HD)))
    assert torch.equal(rows[:, 4:4 + H * HD].unflatten(1, (H, HD)), core.rope(views[0], pos, r))
    assert (rows[:, :4] == 5).all() and (rows[:, 4 + H * HD:] == 5).all()


def test_rope_outside_the_tables_and_non_finite(gpu):
    import torch
    from webpytorch_amd import core
    r = core.Rope(*angles(torch, 10, 32), False)
    x = torch.randn((5, 2, 64)).cuda()
    x[:, :, 40] = math.inf
    x[:, :, 41] = math.nan
    y = core.rope(x, torch.tensor([-1, 0, 9, 10, 2 ** 31 - 1], dtype=torch.int32).cuda(), r)
    assert (y[[0, 3, 4]] == 0).all() and torch.isinf(y[1:3, :, 40]).all() and torch.isnan(y[1:3, :, 41]).all()
    assert torch.equal(y[1, :, :40], x[1, :, :40]) and torch.isfinite(y[2, :, :40]).all()


@pytest.mark.parametrize("pairs", [False, True])
def test_rope_gradient(gpu, pairs):
    """The transposed rotation is the gradient: against differences, and with the forward one (x R y = y R^T x)."""
    import torch
    from webpytorch_amd import core
    g = torch.Generator().manual_seed(11)
    T, H, HD, rot = 4, 2, 64, 48
    r = core.rope_tables(64, rot, scaling={"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 16}, interleaved=pairs)
    x, dy = (torch.randn((T, H, HD), generator=g).cuda() for _ in range(2))
    pos = torch.tensor([0, 7, 33, 63], dtype=torch.int32).cuda()
    dx = core.rope(dy, pos, r, transpose=True).double()
    assert abs(float((core.rope(x, pos, r).double() * dy.double()).sum() - (x.double() * dx).sum())) < 1e-4
    for at in [(0, 0, 0), (1, 1, 5), (2, 0, 40), (3, 1, 47), (3, 0, 60)]:
        up, down = x.clone(), x.clone()
        up[at] += 0.5  # the rotation is linear: differences of any width are exact but for rounding
        down[at] -= 0.5
        diff = ((core.rope(up, pos, r).double() - core.rope(down, pos, r).double()) * dy.double()).sum()
        assert abs(float(diff - dx[at])) < 1e-5 * float(dy.abs().max()) * 8


def test_rope_rotates_as_the_decoder_does(gpu):
    """Half layout over the whole head with the plain tables: `qk_norm_rope`'s rotation, to the rounding of its products."""
    import torch
    from webpytorch_amd import core
    T, NH, NKV, HD = 6, 4, 2, 64
    qkv = torch.randn((T, (NH + 2 * NKV) * HD)).cuda()
    r = core.rope_tables(64, HD, theta=1e6)
    kc, vc = (torch.zeros((NKV, 64, HD), device="cuda") for _ in range(2))
    q = core.qk_norm_rope(qkv, torch.tensor([20], dtype=torch.int32).cuda(), r.cos, r.sin, NH, (kc, vc))
    mine = core.rope(qkv[:, :NH * HD].unflatten(1, (NH, HD)), torch.arange(20, 20 + T, dtype=torch.int32).cuda(), r)
    assert float((q - mine).abs().max()) < 4 * U32 * float(qkv.abs().max()) * 2


def make(torch, seed, S, NH, NKV, HD, P, x, cache, lens, T, extra=2):
    """Rows, positions (lens[s] tokens are there, then T new ones) and a page table in random order over a random cache."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-(n + T) // P) for n in lens]
    num, most = sum(need) + extra, max(need)
    order = torch.randperm(num, generator=g).to(torch.int32)
    pages, at = torch.full((S, most), -1, dtype=torch.int32), 0
    for s, n in enumerate(need):
        pages[s, :n] = order[at:at + n]
        at += n
    c = torch.randn((num, 2, NKV, P, HD), generator=g).to(getattr(torch, cache))
    qkv = (torch.randn((S, T, (NH + 2 * NKV) * HD), generator=g) * 2).to(getattr(torch, x))
    pos = torch.tensor(lens, dtype=torch.int32)[:, None] + torch.arange(T, dtype=torch.int32)[None]
    return qkv, pos, pages, c


@pytest.mark.parametrize("x,cache", [("float32", "float16"), ("float16", "float16"), ("float32", "float32"), ("float16", "float32")])
@pytest.mark.parametrize("NH,NKV,HD,P,rot,pairs,norm", [
    (4, 2, 64, 16, 64, False, "qk"), (7, 1, 128, 32, 64, True, ""), (3, 3, 192, 16, 192, False, "q"), (4, 1, 256, 64, 128, True, "k"),
    (14, 2, 64, 128, 20, False, "qk"), (0, 2, 128, 16, 128, False, "k"), (5, 5, 64, 16, 0, False, "qk"), (2, 1, 192, 32, 6, True, "qk")])
@pytest.mark.parametrize("T", [1, 3, 50])
def test_append(gpu, NH, NKV, HD, P, rot, pairs, norm, T, x, cache):
    """Queries, written slots, and every other slot as it was."""
    import torch
    from webpytorch_amd import core
    lens = [0, P - 1, P, 2 * P + 5]
    qkv, pos, pages, c = make(torch, HD + T, 4, NH, NKV, HD, P, x, cache, lens, T)
    pos[1, T // 2:] = -1  # fewer tokens
    pages[2, -1] = -1     # pages that are missing, and one outside the cache
    pages[3, 2] = c.shape[0]
    rows = lens[3] + T - 1  # the last position lies behind the tables
    r = None if rot == 0 else core.Rope(*angles(torch, rows, rot), pairs)
    qn, kn = (torch.randn(HD).cuda() if n in norm else None for n in "qk")
    dev = c.cuda()
    got = core.paged_append(qkv.cuda(), pos.cuda(), pages.cuda(), dev, NH, r, qn=qn, kn=kn, eps=1e-5)
    cpu = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    q, full, qm, cm, written = paged.append(qkv.numpy(), pos.numpy(), pages.numpy(), c.numpy(), NH, None if r is None else (cpu(r.cos), cpu(r.sin), pairs),
                                   cpu(qn), cpu(kn), 1e-5)
    assert got.shape == (4, T, NH, HD) and got.dtype == qkv.dtype
    near(got, q, qm, NORMED, x == "float16")
    near(dev, full, cm, NORMED, cache == "float16")
    dev, written = dev.cpu(), torch.from_numpy(written)[:, None, None, :, None].expand(c.shape)
    assert torch.equal(dev[~written], c[~written])
    assert torch.equal(dev[:, 1][written[:, 1]], torch.from_numpy(full).to(c.dtype)[:, 1][written[:, 1]])  # values as they are


def test_append_long_prompt_of_strided_rows(gpu):
    """Many heads a thread, rows within wider ones."""
    import torch
    from webpytorch_amd import core
    qkv, pos, pages, c = make(torch, 3, 2, 8, 2, 128, 64, "float32", "float16", [0, 37], 900)
    r = core.Rope(*angles(torch, 1000, 128), False)
    wide = torch.randn((2, 900, qkv.shape[2] + 64)).cuda()
    wide[..., :qkv.shape[2]] = qkv.cuda()
    a, b = c.cuda(), c.cuda()
    qa = core.paged_append(qkv.cuda(), pos.cuda(), pages.cuda(), a, 8, r)
    qb = core.paged_append(wide[..., :qkv.shape[2]], pos.cuda(), pages.cuda(), b, 8, r)
    assert torch.equal(qa, qb) and torch.equal(a, b)
    q, full, qm, cm, _ = paged.append(qkv.numpy(), pos.numpy(), pages.numpy(), c.numpy(), 8, (r.cos.cpu().numpy(), r.sin.cpu().numpy(), False))
    near(qa, q, qm, ROTATED, False)
    near(a, full, cm, ROTATED, True)
    odd = torch.empty(qkv.numel() + 1).cuda()[1:].view(qkv.shape).copy_(qkv)  # rows that start off 16 bytes
    qc = core.paged_append(odd, pos.cuda(), pages.cuda(), c.cuda(), 8, r)
    assert torch.equal(qa, qc)


@pytest.mark.parametrize("scaling", [None, {"type": "linear", "factor": 8.0},
                                     {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 500},
                                     {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 64},
                                     {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 256, "attention_factor": 1.5},
                                     {"rope_type": "wavelength", "factor": 8.0, "original_max_position_embeddings": 128}])
def test_tables(gpu, scaling):
    import torch
    from webpytorch_amd import core
    n, rot, theta = 1024, 64, 1e4
    r = core.rope_tables(n, rot, theta, scaling)
    plain = np.array([theta ** (-2 * i / rot) for i in range(rot // 2)])
    f, m = plain.copy(), 1.0
    if scaling:
        k, F, orig = scaling.get("rope_type", scaling.get("type")), scaling["factor"], scaling.get("original_max_position_embeddings")
        if k == "linear":
            f = plain / F
        elif k == "dynamic":
            base = theta * (F * n / orig - (F - 1)) ** (rot / (rot - 2))
            f = np.array([base ** (-2 * i / rot) for i in range(rot // 2)])
        elif k == "yarn":
            i_of = lambda turns: rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
            lo, hi = max(math.floor(i_of(32)), 0), min(math.ceil(i_of(1)), rot - 1)
            for i in range(rot // 2):
                w = min(max((i - lo) / (hi - lo), 0), 1)
                f[i] = plain[i] * (1 - w) + plain[i] / F * w
            m = scaling.get("attention_factor", 0.1 * math.log(F) + 1)
        else:
            for i in range(rot // 2):
                wave = 2 * math.pi / plain[i]
                if wave > orig:
                    f[i] = plain[i] / F
                elif wave >= orig / 4:
                    w = (orig / wave - 1) / 3
                    f[i] = (1 - w) * plain[i] / F + w * plain[i]
    a = np.arange(n)[:, None] * f[None, :]
    # fp64 angles to 1e-13 of their size, one rounding to fp32
    for t, want in ((r.cos, np.cos(a) * m), (r.sin, np.sin(a) * m)):
        assert np.abs(t.cpu().numpy() - want).max() <= U32 * 2 * abs(m) + 1e-12 * n
    assert r.cos.dtype == torch.float32 and tuple(r.cos.shape) == (n, rot // 2)
