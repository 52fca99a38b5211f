"""GPU: what `score` leaves behind, and the workspace of prompts through layers off the matrix cores."""
import pytest

from webpytorch_amd import synth

pytestmark = pytest.mark.gpu

SMALL = dict(L=1, H=256, NH=4, NKV=2, HD=64, I=512, V=2048, gs=128, bits=4)


def model(w, lmax, **kw):
    from webpytorch_amd import llm
    return llm.CausalLM.from_weights(w, lmax=lmax, **kw)


@pytest.mark.parametrize("kv_bits", [None, 4])
def test_score_leaves_the_sequence_reset(gpu, kv_bits, monkeypatch):
    """After a text of several pieces, and after an error between two of them."""
    from webpytorch_amd import core, llm
    monkeypatch.setattr(llm.CausalLM, "PREFILL_ROWS", 16)
    ids = [int(i) for i in synth.prompt_ids(41, 40, SMALL["V"])]
    m = model(synth.decoder_weights(41, **SMALL), 64, kv_bits=kv_bits)
    m.score(ids)
    assert not m.state.any()
    calls, run = [], core.token_logprobs

    def second_fails(*a):
        calls.append(0)
        if len(calls) == 2:
            raise RuntimeError("planted")
        return run(*a)
    monkeypatch.setattr(core, "token_logprobs", second_fails)
    with pytest.raises(RuntimeError, match="planted"):
        m.score(ids)
    assert not m.state.any()


def test_score_keeps_no_buffers_of_alternatives(gpu):
    """The rows that `generate(logprobs=k)` keeps for its graphs are not made for `score`, whose results are its own."""
    ids = [int(i) for i in synth.prompt_ids(42, 20, SMALL["V"])]
    m = model(synth.decoder_weights(42, **SMALL), 64)
    assert m.score(ids, 7).top_ids.shape == (19, 7)
    for bad in (33, -1):
        with pytest.raises(ValueError, match="alternatives"):
            m.score(ids, bad)
    assert not m._lp_rows


def test_layers_off_the_matrix_cores_have_their_workspace_from_the_start(gpu):
    """A zero offset that is no whole number keeps a prompt's products on the GEMV, whose sums of many rows are more
    than the matrix-core product takes: all allocated with the engine, none during a prompt."""
    from webpytorch_amd import core
    sh = dict(SMALL, H=1024, NH=16, I=9728)
    w = synth.decoder_weights(43, **sh)
    for lay in w["layers"]:
        for name in ("q", "k", "v", "o", "gate", "up", "down"):
            lay[name]["zoff"] = 0.5
    m = model(w, 520, persistent=False)
    ids = [int(i) for i in synth.prompt_ids(43, 500, sh["V"])]
    m.generate(ids[:20], 2)  # the first-use checks have the stream's workspace
    before = {k: t.numel() for k, t in core._WORKSPACE.items()}
    for n in (100, 333, 500):
        m.generate(ids[:n], 2)
    assert {k: t.numel() for k, t in core._WORKSPACE.items()} == before


def test_rows_past_the_gemvs_workspace_go_in_pieces(gpu, monkeypatch):
    """The products of the test above with 16 MB for them: a prompt of 500 rows takes several calls, and no more memory."""
    from webpytorch_amd import core
    sh = dict(SMALL, H=1024, NH=16, I=9728)
    w = synth.decoder_weights(43, **sh)
    for lay in w["layers"]:
        for name in ("q", "k", "v", "o", "gate", "up", "down"):
            lay[name]["zoff"] = 0.5
    ids = [int(i) for i in synth.prompt_ids(43, 500, sh["V"])]
    a = model(w, 520, persistent=False)
    monkeypatch.setattr(core, "GEMV_ROWS_BYTES", 16 << 20)
    b = model(w, 520, persistent=False)
    assert b.ws.numel() <= 16 << 20 < a.ws.numel()
    for m in (a, b):
        m.generate(ids[:20], 2)
    before = {k: t.numel() for k, t in core._WORKSPACE.items()}
    for n in (9, 100, 500):
        la, lb = [(m.generate(ids[:n], 1), m.buf["logits"].clone())[1] for m in (a, b)]
        assert float((la - lb).norm()) <= 1e-5 * float(la.norm())
    assert {k: t.numel() for k, t in core._WORKSPACE.items()} == before
