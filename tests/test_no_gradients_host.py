"""Operators without a backward refuse inputs that want one, rather than give
outputs that are cut off from them."""
import pytest
import torch

from specfit_amd import ops
from specfit_amd.rotary import RotaryTable, rotary_frequencies


def _calls(wants):
    x = torch.zeros((1, 3, 2, 64), requires_grad=wants)
    plain = torch.zeros((1, 3, 2, 64))
    table, positions = rotary_frequencies(64), torch.arange(3)
    logits = torch.zeros((2, 7), requires_grad=wants)
    return {
        "kv_append key": lambda: ops.kv_append(None, 0, x, plain, 0),
        "kv_append value": lambda: ops.kv_append(None, 0, plain, x, 0),
        "block_attention": lambda: ops.block_attention(None, 0, x, 3, None, 1.0),
        "rotary_embed q": lambda: ops.rotary_embed(x, plain, positions, table),
        "rotary_embed k": lambda: ops.rotary_embed(plain, x, positions, table),
        "adjust_logits": lambda: ops.adjust_logits(logits),
        "adjust_logits bias": lambda: ops.adjust_logits(logits.detach(),
                                                        bias=torch.zeros(7, requires_grad=wants)),
    }


@pytest.mark.parametrize("name", _calls(False))
def test_inputs_that_want_a_gradient(name):
    with pytest.raises(ValueError, match="no gradient"):
        _calls(True)[name]()
    with torch.no_grad(), pytest.raises((ValueError, AttributeError)) as next_check:
        _calls(True)[name]()
    assert "gradient" not in str(next_check.value)
    with pytest.raises((ValueError, AttributeError)) as next_check:
        _calls(False)[name]()
    assert "gradient" not in str(next_check.value)


def test_greedy_tokens_have_none_to_lose():
    with pytest.raises(ValueError, match="device"):
        ops.greedy_tokens(torch.zeros((2, 7), requires_grad=True))


def test_a_layer_with_a_rotary_table():
    """Batches and head dims whose rotary embedding torch differentiated before."""
    from transformers import Qwen3MoeConfig
    from transformers.models.qwen3_moe.modeling_qwen3_moe import Qwen3MoeAttention

    from specfit_amd.runtime.qwen3_attention import Qwen3AttentionHip

    config = Qwen3MoeConfig(vocab_size=64, hidden_size=32, num_attention_heads=4, head_dim=64,
                            num_key_value_heads=2, num_hidden_layers=1,
                            attn_implementation="eager")
    hidden = torch.randn((2, 5, 32), requires_grad=True)
    rotary = torch.ones((2, 5, 64)), torch.zeros((2, 5, 64))
    ids = torch.arange(5)[None]
    module = Qwen3AttentionHip.from_module(Qwen3MoeAttention(config, layer_idx=0))
    module(hidden, rotary, None, position_ids=ids)[0].sum().backward()
    assert hidden.grad.any()
    module.rotary = RotaryTable(64, 64, False, 1.0, torch.zeros(32, dtype=torch.float64))
    with pytest.raises(ValueError, match="no gradient"):
        module(hidden, rotary, None, position_ids=ids)
