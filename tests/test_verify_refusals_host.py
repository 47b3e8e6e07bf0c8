"""What a verification step refuses before its forward, and what a refused layer
leaves behind; on the CPU, with stand-ins for the device side."""
import pytest
import torch

from specfit_amd.runtime import Eagle3DraftTree, LogitRules, verify_draft_tree


class _Cache:
    def get_seq_length(self, layer=0):
        return 5


def _no_forward(**kwargs):
    raise AssertionError("the forward was reached")


@pytest.mark.parametrize("more", ({}, dict(commit=False), dict(rules=LogitRules()),
                                  dict(allowed=torch.zeros((1, 4), dtype=torch.int32))))
def test_a_seed_that_is_no_token(more):
    """-1 is the pending seed where nothing was allowed: also a call without rules
    refuses it, before it can index the embedding."""
    tree = Eagle3DraftTree((), (), (), (), ())
    with pytest.raises(ValueError, match="seed"):
        verify_draft_tree(_no_forward, tree, torch.tensor([[-1]]), _Cache(), **more)
    with pytest.raises(ValueError, match="shape"):
        verify_draft_tree(_no_forward, tree, torch.tensor([-1, 3]), _Cache(), **more)
    with pytest.raises(AssertionError, match="forward"):
        verify_draft_tree(_no_forward, tree, torch.tensor([[0]]), _Cache(), **more)


def _layer(monkeypatch, refuse):
    from test_block_cache_host import _Calls
    from transformers import Qwen3MoeConfig
    from transformers.models.qwen3_moe.modeling_qwen3_moe import Qwen3MoeAttention

    from specfit_amd.runtime import BlockKVCache, block_kv_cache
    from specfit_amd.runtime.qwen3_attention import Qwen3AttentionHip

    _Calls().install(monkeypatch)

    def attention(blocks, layer, query, keys, mask, scale):
        if refuse:
            raise TypeError("block attention takes a bool mask (True = attend)")
        return torch.zeros((query.shape[0], query.shape[2], query.shape[1], query.shape[3]))
    block_kv_cache.ops.block_attention = attention
    config = Qwen3MoeConfig(vocab_size=64, hidden_size=32, num_attention_heads=4, head_dim=64,
                            num_key_value_heads=2, num_hidden_layers=3)
    torch.manual_seed(0)
    module = Qwen3AttentionHip.from_module(Qwen3MoeAttention(config, layer_idx=1)).eval()
    return module, BlockKVCache(3, 2, 64, 200)


@torch.no_grad()
def test_a_refused_attention_leaves_the_cache_as_it_was(monkeypatch):
    module, cache = _layer(monkeypatch, refuse=True)
    for layer in range(3):
        cache.append(layer, torch.zeros((1, 2, 70, 64)), torch.zeros((1, 2, 70, 64)))
    cache.commit()
    hidden, rotary = torch.randn((1, 5, 32)), (torch.ones((1, 5, 64)), torch.zeros((1, 5, 64)))
    with pytest.raises(TypeError, match="bool"):
        module(hidden, rotary, torch.zeros((1, 1, 5, 75)), past_key_values=cache)
    assert [cache.get_seq_length(l) for l in range(3)] == [70, 70, 70]
    module, cache = _layer(monkeypatch, refuse=False)
    module(hidden, rotary, None, past_key_values=cache)
    assert [cache.get_seq_length(l) for l in range(3)] == [0, 5, 0]
    cache.crop(3, layer=1)
    cache.append(2, torch.zeros((1, 2, 9, 64)), torch.zeros((1, 2, 9, 64)))
    cache.crop(-1, layer=2)
    assert [cache.get_seq_length(l) for l in range(3)] == [0, 3, 8]
    with pytest.raises(IndexError):
        cache.crop(0, layer=3)
