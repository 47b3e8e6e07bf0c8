"""Rotary frequencies against transformers' (fp32) ones, and their refusals."""
import math

import pytest
import torch

from specfit_amd.rotary import RotaryTable, rotary_frequencies


def _config(parameters, **kwargs):
    from transformers import Qwen3MoeConfig
    return Qwen3MoeConfig(**{**dict(num_attention_heads=4, num_key_value_heads=2, head_dim=128,
                                    hidden_size=64, max_position_embeddings=40960,
                                    rope_parameters=parameters), **kwargs})


@pytest.mark.parametrize("parameters,seq_len", [
    ({"rope_type": "default"}, None),
    ({"rope_type": "linear", "factor": 4.0}, None),
    ({"rope_type": "dynamic", "factor": 2.0}, 100000),
    ({"rope_type": "dynamic", "factor": 2.0}, 100),
    ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
      "original_max_position_embeddings": 8192}, None),
    ({"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}, None),
    ({"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096,
      "mscale": 1.0, "mscale_all_dim": 0.707, "beta_fast": 16, "beta_slow": 2}, None),
    ({"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768,
      "truncate": False, "attention_factor": 1.25}, None),
    ({"rope_type": "longrope", "short_factor": [1.0 + i / 64 for i in range(64)],
      "long_factor": [2.0 + i for i in range(64)], "factor": 8.0,
      "original_max_position_embeddings": 4096}, 10000),
    ({"rope_type": "longrope", "short_factor": [1.0 + i / 64 for i in range(64)],
      "long_factor": [2.0 + i for i in range(64)], "factor": 8.0,
      "original_max_position_embeddings": 4096}, 100)])
def test_frequencies_of_a_config(parameters, seq_len):
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    from transformers.models.qwen3_moe.modeling_qwen3_moe import Qwen3MoeRotaryEmbedding

    config = _config({**parameters, "rope_theta": 1e6})
    kind = parameters["rope_type"]
    if kind == "default":
        want, factor = Qwen3MoeRotaryEmbedding.compute_default_rope_parameters(config)
    else:
        want, factor = ROPE_INIT_FUNCTIONS[kind](config, "cpu", seq_len=seq_len)
    table = RotaryTable.from_config(config, seq_len=seq_len)
    assert table.turns.dtype == torch.float64 and table.turns.shape == (64,)
    assert not table.interleaved and table.rotary_dim == 128
    # transformers rounds the exponent, the power and the blends to fp32: the power
    # of 10^6 turns an exponent's 2^-24 into 14 2^-24.
    assert torch.allclose(table.turns * 2 * math.pi, want.double(), rtol=32 * 2.0 ** -24, atol=0)
    assert table.factor == pytest.approx(factor, rel=1e-6)


def test_plain_frequencies():
    table = rotary_frequencies(8, base=100.0, rotary_dim=4, interleaved=True)
    assert table.interleaved and table.factor == 1.0
    assert (table.turns * 2 * math.pi).tolist() == pytest.approx([1.0, 0.1], rel=1e-15)
    partial = RotaryTable.from_config(_config({"rope_type": "default", "rope_theta": 1e4,
                                               "partial_rotary_factor": 0.25}))
    assert partial.rotary_dim == 32 and partial.head_dim == 128


def test_refusals():
    for kwargs in (dict(rotary_dim=3), dict(rotary_dim=66), dict(rotary_dim=0), dict(base=1.0),
                   dict(scaling={"rope_type": "other"}), dict(scaling={"rope_type": "yarn", "factor": 2.0}),
                   dict(scaling={"rope_type": "dynamic", "factor": 2.0}),
                   dict(scaling={"rope_type": "longrope", "short_factor": [1.0],
                                 "long_factor": [1.0], "original_max_position_embeddings": 16})):
        with pytest.raises(ValueError):
            rotary_frequencies(64, **kwargs)
