"""Models that stretch or part-rotate their positions (CPU): the decoder's tables are plain, and loading says so."""
import json
import warnings

import pytest

from test_checkpoint import write_gguf
from webpytorch_amd import checkpoint

BASE = {"hidden_size": 96, "num_hidden_layers": 2, "num_attention_heads": 4, "num_key_value_heads": 2, "intermediate_size": 64, "vocab_size": 50,
        "quantization_config": {"bits": 4, "group_size": 32}}


def load(tmp_path, **more):
    with open(tmp_path / "config.json", "w") as f:
        json.dump(dict(BASE, **more), f)
    with warnings.catch_warnings(record=True) as said:
        warnings.simplefilter("always")
        shape, _, _ = checkpoint.gptq_config(str(tmp_path))
    return shape, [str(w.message) for w in said]


@pytest.mark.parametrize("key,value", [("rope_scaling", {"rope_type": "llama3", "factor": 8.0}), ("rope_scaling", {"type": "linear", "factor": 2.0}),
                                       ("partial_rotary_factor", 0.5)])
def test_a_configuration_that_is_not_followed(tmp_path, key, value):
    plain, none = load(tmp_path)
    shape, said = load(tmp_path, **{key: value})
    assert shape == plain and not none
    assert len(said) == 1 and key in said[0]


@pytest.mark.parametrize("more", [{"rope_scaling": None}, {"rope_scaling": "none"}, {"rope_scaling": {"type": "default"}}, {"partial_rotary_factor": 1.0},
                                  {"rope_scaling": {"rope_type": "default", "mrope_section": [16, 24, 24], "type": "mrope"}}])
def test_plain_positions(tmp_path, more):
    assert load(tmp_path, **more)[1] == []


@pytest.mark.parametrize("kvs,tensors,text", [
    ([], [], None), ([("llama.rope.scaling.type", 8, "none")], [], None), ([("llama.rope.scaling.type", 8, "yarn")], [], "yarn"),
    ([("llama.rope.scaling.factor", 6, 4.0)], [], "factor"), ([("llama.rope.scaling.factor", 6, 1.0)], [], None),
    ([("llama.rope.scale_linear", 6, 2.0)], [], "scale_linear"), ([], [("rope_freqs.weight", [1], 0, b"\0\0\0\0")], "rope_freqs")])
def test_gguf(tmp_path, kvs, tensors, text):
    path = str(tmp_path / "m.gguf")
    write_gguf(path, [("general.architecture", 8, "llama")] + kvs, tensors + [("vec", [1], 0, b"\0\0\0\0")])
    with warnings.catch_warnings(record=True) as said:
        warnings.simplefilter("always")
        checkpoint.warn_gguf_positions(checkpoint.GGUFFile(path), "llama.")
    assert [text in str(w.message) for w in said] == ([] if text is None else [True])
