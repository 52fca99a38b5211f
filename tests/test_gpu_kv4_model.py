"""GPU: the decoder with a 4-bit key-value cache, and its log probabilities."""
import numpy as np
import pytest

from oracle import decode, kv4
from webpytorch_amd import synth

pytestmark = pytest.mark.gpu

SMALL = dict(L=2, H=256, NH=4, NKV=2, HD=64, I=512, V=2048, gs=128, bits=4)
WIDE = dict(L=2, H=256, NH=6, NKV=2, HD=128, I=512, V=2048, gs=128, bits=4)
MOE = dict(SMALL, n_experts=8, moe_I=128, top_k=2, qk_norm=True)
# Two passes of the engine over one text (a prompt at once, or token by token) give keys and values that differ
# in their last bits, so that a code in about 10^5 falls on the other side of a border: a step, a quarter of
# a value's spread, in one value of one position. In a model of one layer that moves one score by 0.25 / sqrt(HD)
# = 0.03 (that position's p, 1 / 40 or less, by 3 %), or one dimension of one value that p weighs: 10^-3 of the
# attention's output, and no more of the logits. (Layers on top would turn it into codes of their own.)
MODEL_REL = 5e-3
ORACLE_REL = 2e-4  # the engine's products against the oracle's, 2^-22 of each row's largest value, through two layers


class Kv4Oracle(decode.Qwen2Oracle):
    """Attends over the rows that the engine's caches stand for, after checking that each is within half a
    step (and the roundings of S, Z and the value) of the row it computes itself."""

    def attend(self, q, K, V, mask, scale):
        i = self.layer = (getattr(self, "layer", -1) + 1) % self.L
        rows = []
        for x, (c, S, Z) in zip((K, V), self.caches[i]):
            n = x.shape[1]
            got = kv4.stands_for(c[:, :n], S[:, :n], Z[:, :n])
            S, Z = (np.repeat(np.abs(t[:, :n].astype(np.float64)), 32, -1) for t in (S, Z))
            assert (np.abs(got - x) <= S / 32 + 2.0 ** -10 * (2 * S + Z) + 1e-4 * np.abs(x).max()).all()
            rows.append(got.astype(np.float32))
        return super().attend(q, rows[0], rows[1], mask, scale)


def model(w, lmax, **kw):
    from webpytorch_amd import llm
    return llm.CausalLM.from_weights(w, lmax=lmax, **kw)


@pytest.mark.parametrize("sh", [SMALL, WIDE, MOE], ids=["64", "128", "moe-qk-norm"])
def test_logits_match_the_oracle_over_the_same_cache(gpu, sh):
    w = synth.decoder_weights(21, gaussian=True, **sh)
    ids = synth.prompt_ids(21, 37, sh["V"])
    m = model(w, 64, kv_bits=4)
    tokens = m.generate(ids, 4, use_graph=False).tokens
    o = Kv4Oracle(w, lmax=64)
    o.caches = [kv4.unpack(c.cpu().numpy(), 40) for c in m.kv4]
    cache, pos, step = [None] * o.L, 0, [int(i) for i in ids]
    for n in range(1, 5):
        _, want = o.forward(step, pos, cache)
        assert m.generate(ids, n, use_graph=False).tokens == tokens[:n]
        lg = m.buf["logits"][0].cpu().numpy()
        assert np.linalg.norm(lg - want) <= ORACLE_REL * np.linalg.norm(want)
        pos, step = pos + len(step), tokens[n - 1:n]


@pytest.mark.parametrize("sh", [SMALL, MOE], ids=["dense", "moe-qk-norm"])
@pytest.mark.parametrize("kv_bits", [None, 4])
def test_graphs_eager_steps_and_scores_agree(gpu, sh, kv_bits):
    """Captured steps give the eager ones' bits, log probabilities too; scoring the whole text in one pass gives
    the same to the products' rounding (4 bits: MODEL_REL of the logits)."""
    import torch
    sh = dict(sh, L=1) if kv_bits == 4 else sh
    w = synth.decoder_weights(22, gaussian=True, **sh)
    ids = [int(i) for i in synth.prompt_ids(22, 40, sh["V"])]
    a, b = model(w, 96, kv_bits=kv_bits), model(w, 96, kv_bits=kv_bits)
    plain = a.generate(ids, 24)
    ra, rb = a.generate(ids, 24, logprobs=5), b.generate(ids, 24, use_graph=False, logprobs=5)
    assert plain.logprobs is None and plain.tokens == ra.tokens == rb.tokens
    for x, y in zip(ra.logprobs, rb.logprobs):
        assert x.shape[0] == 24 and torch.equal(x, y)
    again = a.generate(ids, 24, logprobs=5)
    assert all(torch.equal(x, y) for x, y in zip(again.logprobs, ra.logprobs))
    assert ra.logprobs.top_ids[:, 0].tolist() == ra.tokens and ra.logprobs.ranks.tolist() == [0] * 24
    assert torch.equal(ra.logprobs.top_logprobs[:, 0], ra.logprobs.logprobs)
    s = a.score(ids + ra.tokens, 5)
    assert s.logprobs.shape == (63,) and s.top_ids.shape == (63, 5)
    size = float(a.buf["logits"].norm())
    tol = MODEL_REL * size if kv_bits == 4 else 1e-3
    assert float((s.logprobs[39:] - ra.logprobs.logprobs).abs().max()) < tol
    assert float((s.entropy[39:] - ra.logprobs.entropy).abs().max()) < 10 * tol
    assert a.generate(ids, 24).tokens == plain.tokens


def test_score_in_several_chunks(gpu):
    """More rows than one chunk of logits holds, against token by token (each prompt one longer)."""
    w = synth.decoder_weights(23, gaussian=True, **SMALL)
    ids = [int(i) for i in synth.prompt_ids(23, 60, SMALL["V"])]
    m = model(w, 64)
    whole = m.score(ids, 3)
    m.SCORE_ROWS = 25
    parts = m.score(ids, 3)
    for x, y in zip(whole, parts):
        assert x.shape == y.shape and np.allclose(x.cpu().numpy(), y.cpu().numpy(), rtol=0, atol=1e-3)
    for n in (1, 26, 59):
        m.generate(ids[:n], 1)
        lg = m.buf["logits"][0].double().cpu().numpy()
        want = lg[ids[n]] - lg.max() - np.log(np.exp(lg - lg.max()).sum())
        assert abs(float(whole.logprobs[n - 1]) - want) < 1e-3


def test_fused_and_plain_steps_agree(gpu):
    w = synth.decoder_weights(24, gaussian=True, **dict(WIDE, L=1))
    ids = synth.prompt_ids(24, 33, WIDE["V"])
    a, b = model(w, 64, kv_bits=4), model(w, 64, kv_bits=4, fused=False)
    for m in (a, b):
        m.generate(ids, 2, use_graph=False)
    la, lb = a.buf["logits"], b.buf["logits"]
    assert float((la - lb).norm()) <= MODEL_REL * float(lb.norm())
    # the same prompt pass, so the same cache
    assert all(np.array_equal(x[:, 0].cpu().numpy(), y[:, 0].cpu().numpy()) for x, y in zip(a.kv4, b.kv4))


def test_context_past_the_fp32_attention(gpu):
    """20000 positions: the token behind a prompt of 17000 is that of the prompt one longer."""
    sh = dict(SMALL, L=1)
    w = synth.decoder_weights(25, gaussian=True, **sh)
    ids = [int(i) for i in synth.prompt_ids(25, 17000, sh["V"])]
    m = model(w, 20000, kv_bits=4)
    two = m.generate(ids, 2, use_graph=False).tokens
    one = m.buf["logits"].clone()
    m.generate(ids + two[:1], 1)
    assert float((m.buf["logits"] - one).norm()) <= MODEL_REL * float(one.norm())


@pytest.mark.parametrize("kv_bits", [None, 4])
def test_prompts_in_pieces(gpu, kv_bits, monkeypatch):
    """A prompt of several pieces (the last of one token, of some, whole) against the same in one."""
    from webpytorch_amd import llm
    sh = dict(SMALL, L=1)
    w = synth.decoder_weights(32, gaussian=True, **sh)
    ids = [int(i) for i in synth.prompt_ids(32, 48, sh["V"])]
    a = model(w, 64, kv_bits=kv_bits)
    monkeypatch.setattr(llm.CausalLM, "PREFILL_ROWS", 16)
    b = model(w, 64, kv_bits=kv_bits)
    assert b.buf["h"].shape[0] == 16 and b.history.shape[0] == 64
    for n in (15, 16, 17, 33, 40, 48):
        for m in (a, b):
            m.generate(ids[:n], 3, use_graph=False)
        assert int(b.state[0]) == n + 2
        la, lb = a.buf["logits"], b.buf["logits"]
        assert float((la - lb).norm()) <= MODEL_REL * float(la.norm())
    sa, sb = a.score(ids, 2), b.score(ids, 2)
    tol = MODEL_REL * float(la.norm())
    assert sb.logprobs.shape == (47,) and float((sa.logprobs - sb.logprobs).abs().max()) < tol


def test_long_context_of_wide_layers(gpu):
    """40000 positions of a layer of 37888 columns: more rows at a time than its products are made for."""
    sh = dict(SMALL, L=1, I=18944)
    w = synth.decoder_weights(33, gaussian=True, **sh)
    ids = [int(i) for i in synth.prompt_ids(33, 20, sh["V"])]
    a, b = model(w, 40000, kv_bits=4), model(w, 64, kv_bits=4)
    assert a.generate(ids, 5).tokens == b.generate(ids, 5).tokens
    # 16384 rows of 18944 values as two fp16 numbers (1.24e9 bytes), not the GEMV's sums of as many rows (35e9)
    assert a.ws.numel() < 1.3e9


def test_persistent_step_with_logprobs_and_its_timeout(gpu, monkeypatch):
    import torch
    w = synth.decoder_weights(26, gaussian=True, **SMALL)
    ids = synth.prompt_ids(26, 16, SMALL["V"])
    a, b = model(w, 64, persistent=True), model(w, 64, persistent=False)
    ra, rb = a.generate(ids, 9, logprobs=4), b.generate(ids, 9, logprobs=4)
    assert ra.tokens == rb.tokens and torch.equal(ra.logprobs.top_ids[:, 0], rb.logprobs.top_ids[:, 0])
    assert float((ra.logprobs.logprobs - rb.logprobs.logprobs).abs().max()) < 1e-3
    monkeypatch.setenv("MIQ_PD_SPIN_TICKS", "1")
    a._graphs.clear()  # captured now, with the one-tick bound
    with pytest.warns(RuntimeWarning, match="launch sequence"):
        got = a.generate(ids, 9, logprobs=4)
    monkeypatch.delenv("MIQ_PD_SPIN_TICKS")
    assert got.tokens == rb.tokens and a.fallback_steps == 9
    assert all(torch.equal(x, y) for x, y in zip(got.logprobs, rb.logprobs))
    a._graphs.clear()
    assert all(torch.equal(x, y) for x, y in zip(a.generate(ids, 9, logprobs=4).logprobs, ra.logprobs))


@pytest.mark.parametrize("mode", ["native", "requant"])
def test_gguf_model_from_pretrained(gpu, tmp_path, mode):
    """`kv_bits` through the loaders: a GGUF file in its own blocks (the unfused steps) and requantized, a context
    that ends inside a block of the cache."""
    from test_gpu_gguf_model import make_model, oracle_weights
    from webpytorch_amd import llm
    path = tmp_path / "m.gguf"
    mats, floats = make_model(path)[:2]
    m = llm.AutoModelForCausalLM.from_pretrained(str(path), dtype="auto" if mode == "native" else "int4", lmax=45, weights=mode, kv_bits=4)
    ids = [int(i) for i in synth.prompt_ids(31, 37, 2048)]
    tokens = m.generate(ids, 8).tokens
    o = Kv4Oracle(oracle_weights(mats, floats, mode), lmax=64)
    o.caches = [kv4.unpack(c.cpu().numpy(), 45) for c in m.kv4]
    cache, pos, step = [None] * o.L, 0, ids
    for n in range(1, 9):
        _, want = o.forward(step, pos, cache)
        assert m.generate(ids, n).tokens == tokens[:n]
        lg = m.buf["logits"][0].cpu().numpy()
        assert np.linalg.norm(lg - want) <= ORACLE_REL * np.linalg.norm(want)
        pos, step = pos + len(step), tokens[n - 1:n]


def test_score_of_few_rows_needs_the_heads_workspace(gpu):
    """2 to 8 rows of the head split K where one row does not: more workspace than the steps ever take."""
    sh = dict(SMALL, L=1, H=1024, I=256, V=32768)
    m = model(synth.decoder_weights(29, gaussian=True, **sh), 32)
    ids = [int(i) for i in synth.prompt_ids(29, 20, sh["V"])]
    whole = m.score(ids)
    for n in (2, 3, 6, 9):
        got = m.score(ids[:n])
        assert np.allclose(got.logprobs.cpu().numpy(), whole.logprobs[:n - 1].cpu().numpy(), rtol=0, atol=1e-3)


@pytest.mark.parametrize("k", [0, 16, 20, 32])
def test_logprobs_of_a_large_vocabulary(gpu, k):
    """The workspace holds any number of alternatives: of this vocabulary, 16 need more than 32."""
    sh = dict(L=1, H=128, NH=2, NKV=1, HD=64, I=128, V=262144, gs=128, bits=4)
    m = model(synth.decoder_weights(30, gaussian=True, **sh), 16)
    r = m.generate([5, 6, 7], 4, logprobs=k)
    assert r.logprobs.top_ids.shape == (4, k) and r.logprobs.ranks.tolist() == [0] * 4
    if k:
        assert r.logprobs.top_ids[:, 0].tolist() == r.tokens


def test_refusals(gpu):
    w = synth.decoder_weights(27, **SMALL)
    for kw, exc in ((dict(kv_bits=8), ValueError), (dict(kv_bits=4, persistent=True), ValueError)):
        with pytest.raises(exc):
            model(w, 64, **kw)
    small = dict(SMALL, HD=32, NH=8)
    with pytest.raises(NotImplementedError, match="32"):
        model(synth.decoder_weights(28, **dict(small, gs=32)), 64, kv_bits=4)
    m = model(w, 64, kv_bits=4)
    for bad in (33, -1):
        with pytest.raises(ValueError, match="logprobs"):
            m.generate([1, 2], 2, logprobs=bad)
    for ids in ([1], list(range(65))):
        with pytest.raises(ValueError, match="score"):
            m.score(ids)
