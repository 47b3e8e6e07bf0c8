"""The block cache, the rotary table and the rules together, as a
verification loop uses them, on a small offloaded Qwen3-MoE target.

A DynamicCache filled with what the block cache gives back (read) is the same
context for the tree-attention model, so the two paths have to agree to the
roundings of their attention; the tolerance is that of the other model tests
(3e-2 of the largest logit: two bf16 forwards with differently ordered sums)."""
import math

import pytest
import torch

from specfit_amd.rotary import RotaryTable
from specfit_amd.runtime import (TREE_ATTENTION, BlockKVCache, LogitRules, build_offloaded_qwen3,
                                 install_hip_attention, register_tree_attention, synthetic_tree,
                                 verify_draft_tree)

pytestmark = pytest.mark.gpu
VOCAB = 128


def _loaded(device, head_dim=64, layers=2, seed=7):
    from transformers import Qwen3MoeConfig, Qwen3MoeForCausalLM

    torch.manual_seed(seed)
    config = Qwen3MoeConfig(vocab_size=VOCAB, hidden_size=64, intermediate_size=48,
                            moe_intermediate_size=32, num_hidden_layers=layers,
                            num_attention_heads=4, num_key_value_heads=2, head_dim=head_dim,
                            num_experts=4, num_experts_per_tok=2, max_position_embeddings=1024,
                            bos_token_id=1, eos_token_id=2, pad_token_id=0, norm_topk_prob=True)
    model = Qwen3MoeForCausalLM(config).to(torch.bfloat16).eval()
    register_tree_attention()
    model.config._attn_implementation = TREE_ATTENTION
    return build_offloaded_qwen3(model, device=device, slots_per_layer=4)


def _dynamic(cache):
    from transformers import DynamicCache

    other = DynamicCache()
    for layer in range(cache.blocks.layers):
        other.update(*cache.read(layer), layer)
    return other


def _close(a, b):
    a, b = a.float(), b.float()
    torch.testing.assert_close(a, b, atol=3e-2 * b.abs().max().item(), rtol=3e-2)


@pytest.mark.parametrize("head_dim,held", [(64, "e4m3"), (128, "int8")])
@torch.inference_mode()
def test_verification_over_blocks(device, head_dim, held):
    loaded = _loaded(device, head_dim)
    target = loaded.model
    g = torch.Generator().manual_seed(head_dim)
    cache = BlockKVCache.from_config(target.config, 400, held=held, tail_tokens=200, device=device)
    prompt = torch.randint(3, VOCAB, (1, 150), generator=g).to(device)
    out = target(input_ids=prompt, past_key_values=cache, use_cache=True, logits_to_keep=1)
    # Nothing is folded yet: the prompt's forward is the plain model's.
    plain = target(input_ids=prompt, use_cache=False, logits_to_keep=1)
    _close(out.logits, plain.logits)
    assert cache.get_seq_length() == 150
    cache.commit()
    assert cache.folded_tokens == 128
    seed = out.logits.argmax(-1)
    for step in range(8):
        tree = synthetic_tree(24, 4, seed=step, vocab=VOCAB)
        base = cache.get_seq_length()
        other = _dynamic(cache)
        a = verify_draft_tree(target, tree, seed, cache)
        b = verify_draft_tree(target, tree, seed, other, commit=False)
        _close(a.logits, b.logits)
        assert cache.get_seq_length() == base + len(a.verification_positions)
        assert cache.folded_tokens == cache.get_seq_length() // 64 * 64
        assert torch.equal(a.committed, a.verify_ids[:, a.verification_positions])
        # What was kept are the accepted rows (to 8 bits where they folded).
        index = torch.tensor([base + p for p in a.verification_positions], device=device)
        for layer in range(2):
            k, _ = cache.read(layer, max(base, cache.folded_tokens))
            want = other.layers[layer].keys.index_select(2, index)[:, :, -k.shape[2]:] if k.shape[2] else k
            if k.shape[2]:
                _close(k, want)
        seed = a.pending_seed
    # A plain decode step over the same cache.
    nxt = target(input_ids=seed, past_key_values=cache, use_cache=True)
    assert torch.isfinite(nxt.logits.float()).all()
    loaded.close()


@torch.inference_mode()
def test_rules_in_the_verification(device):
    loaded = _loaded(device)
    target = loaded.model
    g = torch.Generator().manual_seed(3)
    prompt = torch.randint(3, VOCAB, (1, 70), generator=g).to(device)
    cache = BlockKVCache.from_config(target.config, 200, held="int8", tail_tokens=128, device=device)
    seed = target(input_ids=prompt, past_key_values=cache, use_cache=True,
                  logits_to_keep=1).logits.argmax(-1)
    cache.commit()
    rules = LogitRules.for_vocab(VOCAB, device, repetition=1.5, presence=0.5, frequency=0.25)
    rules.count(prompt)
    tree = synthetic_tree(12, 3, seed=1, vocab=VOCAB)
    allowed = torch.randint(-2 ** 31, 2 ** 31, (13, 4), generator=g).int()
    allowed[5] = 0
    before = rules.counts.clone()
    result = verify_draft_tree(target, tree, seed, cache, rules=rules, allowed=allowed.to(device))
    # The same by hand, row by row.
    logits, ids = result.logits[0].float().cpu(), result.verify_ids[0].tolist()
    for row, path in enumerate(tree.path_indices()):
        count = before.cpu().double()
        for p in path[path >= 0]:
            count[ids[p]] += 1
        x = logits[row]
        y = torch.where(x < 0, x * 1.5, x / 1.5) - (0.25 * count.float() + 0.5)
        y = torch.where(count > 0, y, x)
        bits = ((allowed[row][:, None] >> torch.arange(32)) & 1).flatten()
        y = torch.where(bits == 0, -math.inf, y)
        want = -1 if row == 5 else int(y.argmax())
        assert int(result.verifier_tokens[0, row]) == want
    counted = before.cpu() + torch.bincount(result.committed.flatten().cpu(), minlength=VOCAB)
    assert torch.equal(rules.counts.cpu(), counted.int())
    # A row in which nothing is allowed ends the path.
    nothing = torch.zeros((13, 4), dtype=torch.int32, device=device)
    result = verify_draft_tree(target, tree, seed, cache, allowed=nothing, commit=False)
    assert result.accepted_node_ids == () and int(result.pending_seed) == -1
    # The sequence ends there.
    length, counted = cache.get_seq_length(), rules.counts.clone()
    for again in (dict(rules=rules), dict(allowed=nothing)):
        with pytest.raises(ValueError, match="seed"):
            verify_draft_tree(target, tree, result.pending_seed, cache, **again)
    assert cache.get_seq_length() == length and torch.equal(rules.counts, counted)
    loaded.close()


@torch.inference_mode()
def test_rotary_from_positions(device):
    """A model whose layers take their rotary embedding from the table agrees
    with the one that uses bf16 cosines; batches and other head dims too."""
    for head_dim, batch in ((128, 1), (64, 3)):
        loaded = _loaded(device, head_dim)
        target = loaded.model
        g = torch.Generator().manual_seed(4)
        ids = torch.randint(3, VOCAB, (batch, 30), generator=g).to(device)
        want = target(input_ids=ids, use_cache=False).logits
        table = RotaryTable.from_config(target.config, device=device)
        assert install_hip_attention(target, rotary=table) == 0  # the layers are there already
        _close(target(input_ids=ids, use_cache=False).logits, want)
        cache = BlockKVCache.from_config(target.config, 64, batch=batch, device=device)
        _close(target(input_ids=ids, past_key_values=cache, use_cache=True).logits, want)
        loaded.close()


@torch.inference_mode()
def test_other_attention_implementations_read_the_cache(device):
    """update() gives plain tensors to attention layers that do not know the
    cache."""
    from transformers import Qwen3MoeConfig, Qwen3MoeForCausalLM

    torch.manual_seed(1)
    config = Qwen3MoeConfig(vocab_size=VOCAB, hidden_size=64, intermediate_size=48,
                            moe_intermediate_size=32, num_hidden_layers=2, num_attention_heads=4,
                            num_key_value_heads=2, head_dim=64, num_experts=4,
                            num_experts_per_tok=2, max_position_embeddings=256)
    model = Qwen3MoeForCausalLM(config).to(torch.bfloat16).to(device).eval()
    ids = torch.randint(3, VOCAB, (1, 40), generator=torch.Generator().manual_seed(2)).to(device)
    cache = BlockKVCache.from_config(config, 100, device=device)
    model(input_ids=ids[:, :33], past_key_values=cache, use_cache=True)
    got = model(input_ids=ids[:, 33:], past_key_values=cache, use_cache=True).logits
    _close(got, model(input_ids=ids, use_cache=False).logits[:, 33:])
    assert cache.get_seq_length() == 40
