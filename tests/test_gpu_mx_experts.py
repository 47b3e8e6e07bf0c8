"""Experts with 4-bit weights (K16) against a 64-bit reference."""
import pytest
import torch

import _mx_reference as ref
from specfit_amd import ops
from specfit_amd.runtime import Qwen3MXExperts

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _case(tokens, hidden, inner, experts, top_k, seed=0, favourite=None, distinct=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.randn((tokens, hidden), generator=g, device=DEV).to(torch.bfloat16)
    packed = (torch.randn((experts, 3 * hidden * inner), generator=g, device=DEV)
              * 1.5 * hidden ** -0.5).to(torch.bfloat16)
    scores = torch.rand((tokens, experts), generator=g, device=DEV)
    if favourite is not None:
        scores[:, favourite] += 1
    index = torch.topk(scores, top_k, dim=1).indices
    if not distinct:
        index = torch.randint(0, experts, (tokens, top_k), generator=g, device=DEV)
    weights = torch.softmax(torch.randn((tokens, top_k), generator=g, device=DEV), 1)
    return h, packed, index, weights.to(torch.bfloat16)


def _check(got, h, index, weights, packed, hidden, inner, **more):
    want, slack = ref.experts(h, index, weights, packed, hidden, inner, **more)
    assert (got.double() - want).abs().le(slack).all()
    if want.norm() > 0:
        # Roundings to 8 bits fall on the other side for a few values only.
        assert (got.double() - want).norm() <= 2.0 ** -7 * want.norm()


SHAPES = [(1, 64, 32, 8, 3), (5, 64, 32, 8, 3), (40, 64, 32, 8, 3), (7, 1000, 424, 20, 2),
          (3, 33, 17, 4, 1), (16, 2048, 768, 16, 8), (17, 2048, 768, 16, 8), (61, 256, 160, 128, 8),
          (150, 256, 96, 4, 2), (300, 512, 256, 6, 2), (1, 4096, 1536, 8, 8), (600, 128, 64, 3, 1),
          (33, 64, 32, 1, 1), (50, 64, 32, 256, 3), (400, 1000, 424, 3, 1), (300, 33, 17, 2, 1),
          (700, 136, 200, 5, 5)]


@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", SHAPES)
def test_experts(tokens, hidden, inner, experts, top_k):
    h, packed, index, weights = _case(tokens, hidden, inner, experts, top_k)
    module = Qwen3MXExperts.from_packed(packed, hidden_size=hidden, intermediate_size=inner)
    _check(module(h, index, weights), h, index, weights, packed, hidden, inner)


@pytest.mark.parametrize("tokens", [20, 200, 700])
def test_a_favourite_takes_every_token(tokens):
    h, packed, index, weights = _case(tokens, 256, 128, 40, 2, favourite=11)
    module = Qwen3MXExperts.from_packed(packed, hidden_size=256, intermediate_size=128)
    _check(module(h, index, weights), h, index, weights, packed, 256, 128)


def test_the_same_expert_twice_and_experts_that_are_not_there():
    h, packed, index, weights = _case(30, 96, 64, 5, 4, distinct=False)
    index[3, 1], index[7], index[9, 2], index[11, 0] = 99, -1, 2 ** 40, 2 ** 32 + 1
    module = Qwen3MXExperts.from_packed(packed, hidden_size=96, intermediate_size=64)
    got = module(h, index, weights)
    _check(got, h, index, weights, packed, 96, 64)
    assert not got[7].any()


def test_a_slot_table_and_rows_that_are_left_alone():
    H, I, E, K = 128, 96, 6, 2
    h, packed, index, weights = _case(50, H, I, E, K)
    records = ops.mx_quantize_experts(packed, H, I)
    slots = torch.zeros((4, records.shape[1]), dtype=torch.uint8, device=DEV)
    table = torch.tensor([2, -1, 0, -1, 3, 1], dtype=torch.int32, device=DEV)
    for e, s in enumerate(table.tolist()):
        if s >= 0:
            slots[s] = records[e]
    plan = ops.dispatch(index, E)
    full = torch.empty((50 * K, H), dtype=torch.bfloat16, device=DEV)
    ops.mx_grouped_swiglu(h, plan, weights.view(-1), records, H, I, full)
    some = torch.full_like(full, 7.0)
    ops.mx_grouped_swiglu(h, plan, weights.view(-1), slots, H, I, some, slot_of_expert=table)
    expert = index.flatten()[plan.perm_pos.long()]
    there = table[expert] >= 0
    assert torch.equal(some[there], full[there]) and (some[~there] == 7).all()


def test_rows_and_tensor_give_the_same_and_no_weights_means_one():
    H, I, E, K = 256, 64, 8, 2
    h, packed, index, _ = _case(12, H, I, E, K)
    records = ops.mx_quantize_experts(packed, H, I)
    plan = ops.dispatch(index, E)
    a, b = (torch.empty((12 * K, H), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    ops.mx_grouped_swiglu(h, plan, None, records, H, I, a)
    ops.mx_grouped_swiglu(ops.mx_quantize(h), plan, None, records, H, I, b)
    ones = torch.ones((12, K), dtype=torch.bfloat16, device=DEV)
    c = torch.empty_like(a)
    ops.mx_grouped_swiglu(h, plan, ones.view(-1), records, H, I, c)
    assert torch.equal(a, b) and torch.equal(a, c)


def test_non_finite_tokens_stay_alone():
    h, packed, index, weights = _case(40, 128, 64, 4, 2)
    h[5, 9], h[17, 100] = float("inf"), float("nan")
    module = Qwen3MXExperts.from_packed(packed, hidden_size=128, intermediate_size=64)
    bad = torch.isnan(module(h, index, weights)).all(1)
    assert bad.nonzero().flatten().tolist() == [5, 17]
    assert not torch.isnan(module(h, index, weights)[~bad]).any()


def test_from_an_hf_module():
    from transformers import Qwen3MoeConfig
    from transformers.models.qwen3_moe.modeling_qwen3_moe import Qwen3MoeExperts

    config = Qwen3MoeConfig(hidden_size=64, moe_intermediate_size=48, num_experts=6)
    hf = Qwen3MoeExperts(config).to(torch.bfloat16).to(DEV)
    with torch.no_grad():
        for p in hf.parameters():
            p.normal_(0, 0.2)
    packed = torch.cat([hf.gate_up_proj.detach().flatten(1), hf.down_proj.detach().flatten(1)], 1)
    ours = Qwen3MXExperts.from_module(hf)
    again = Qwen3MXExperts.from_packed(packed, hidden_size=64, intermediate_size=48)
    assert torch.equal(ours.records, again.records)
    h, _, index, weights = _case(9, 64, 48, 6, 2)
    _check(ours(h, index, weights), h, index, weights, packed, 64, 48)


@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_captured_and_replayed(tokens):
    H, I, E, K = 256, 128, 16, 4
    h, packed, index, weights = _case(tokens, H, I, E, K)
    module = Qwen3MXExperts.from_packed(packed, hidden_size=H, intermediate_size=I)
    h_in, index_in, w_in = h.clone(), index.clone(), weights.clone()
    module(h_in, index_in, w_in)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = module(h_in, index_in, w_in)
    for seed in range(3):
        h, _, index, weights = _case(tokens, H, I, E, K, seed=seed + 5)
        h_in.copy_(h)
        index_in.copy_(index)
        w_in.copy_(weights)
        graph.replay()
        eager = module(h, index, weights)
        assert torch.equal(out, eager)


def test_on_another_stream():
    h, packed, index, weights = _case(33, 128, 64, 6, 2)
    records = ops.mx_quantize_experts(packed, 128, 64)
    plan = ops.dispatch(index, 6)
    want = torch.empty((66, 128), dtype=torch.bfloat16, device=DEV)
    ops.mx_grouped_swiglu(h, plan, weights.view(-1), records, 128, 64, want)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = torch.zeros_like(want)
    side.wait_stream(torch.cuda.current_stream())
    ops.mx_grouped_swiglu(h, plan, weights.view(-1), records, 128, 64, got, stream=side)
    x = h[:, :100]
    w = ops.mx_quantize_weight(torch.randn((40, 100), device=DEV))
    side.wait_stream(torch.cuda.current_stream())
    y = ops.mx_linear(x, w, stream=side)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(y, ops.mx_linear(x, w))


def _routed(h, index, weights, packed, hidden, inner, **more):
    records = ops.mx_quantize_experts(packed, hidden, inner)
    return ops.mx_routed_swiglu(h, index, weights, records, hidden, inner, **more)


@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", SHAPES[:10] + [(3, 2048, 768, 128, 1), (2, 520, 200, 9, 5),
                                                                          (1, 64, 32, 40, 16)])
def test_routed(tokens, hidden, inner, experts, top_k):
    h, packed, index, weights = _case(tokens, hidden, inner, experts, top_k, seed=3)
    got = _routed(h, index, weights, packed, hidden, inner)
    _check(got, h, index, weights, packed, hidden, inner)
    assert torch.equal(got, _routed(ops.mx_quantize(h), index, weights, packed, hidden, inner))


def test_routed_with_a_table_repeats_and_experts_that_are_not_there():
    h, packed, index, weights = _case(9, 96, 64, 5, 4, distinct=False)
    index[3, 1], index[7], index[2, 0], index[1, 3] = 99, -1, 2 ** 40, -2 ** 40
    table = torch.tensor([2, -1, 0, 3, 1], dtype=torch.int32, device=DEV)
    records = ops.mx_quantize_experts(packed, 96, 64)
    slots = torch.zeros((4, records.shape[1]), dtype=torch.uint8, device=DEV)
    slots[table[table >= 0].long()] = records[table >= 0]
    got = ops.mx_routed_swiglu(h, index, weights, slots, 96, 64, slot_of_expert=table)
    there = torch.where(index == 1, -1, index)
    _check(got, h, there, weights, packed, 96, 64)
    assert not got[7].any()
    h[5, 9] = float("nan")
    assert torch.isnan(ops.mx_routed_swiglu(h, index, weights, records, 96, 64)).all(1).tolist() \
        == [i == 5 for i in range(9)]


def test_routed_captured_and_on_another_stream():
    h, packed, index, weights = _case(2, 256, 128, 16, 4)
    records = ops.mx_quantize_experts(packed, 256, 128)
    want = ops.mx_routed_swiglu(h, index, weights, records, 256, 128)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    columns = h.t().contiguous().t()
    side.wait_stream(torch.cuda.current_stream())
    got = ops.mx_routed_swiglu(columns, index, weights, records, 256, 128, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.mx_routed_swiglu(h, index, weights, records, 256, 128)
    for seed in range(3):
        new, _, i2, w2 = _case(2, 256, 128, 16, 4, seed=seed + 5)
        h.copy_(new), index.copy_(i2), weights.copy_(w2)
        graph.replay()
        assert torch.equal(out, ops.mx_routed_swiglu(h, index, weights, records, 256, 128))


@pytest.mark.parametrize("tokens", [2, 12, 90])
def test_one_call_takes_any_rows(tokens):
    H, I, E, K = 128, 64, 6, 3
    h, packed, index, weights = _case(tokens, H, I, E, K)
    records = ops.mx_quantize_experts(packed, H, I)
    want = ops.mx_experts(h, index, weights, records, H, I)
    _check(want, h, index, weights, packed, H, I)
    wide = torch.zeros((tokens, 2 * H + 1), dtype=torch.bfloat16, device=DEV)
    for at in (3, 8, H + 1):
        wide[:, at:at + H] = h
        # Rows rounded here or beforehand: the same codes, so the same bits in one form.
        assert torch.equal(ops.mx_experts(wide[:, at:at + H], index, weights, records, H, I),
                           ops.mx_experts(ops.mx_quantize(h), index, weights, records, H, I))
    columns = h.t().contiguous().t()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = ops.mx_experts(columns, index, weights, records, H, I, stream=side)
    side.synchronize()
    assert torch.equal(got, ops.mx_experts(ops.mx_quantize(h), index, weights, records, H, I))


def test_far_rows():
    """Offsets of rows past 32 bits: the last tokens' outputs are what they are by
    themselves (as many routes to an expert as make the same tiles)."""
    H, I, E, K, T = 2048, 32, 8, 8, 140_000
    h, packed, index, weights = _case(400, H, I, E, K)
    records = ops.mx_quantize_experts(packed, H, I)
    want = ops.mx_experts(h, index, weights, records, H, I)
    many = torch.zeros((T, H), dtype=torch.bfloat16, device=DEV)
    many[-400:] = h
    many_index, many_weights = index.repeat(T // 400, 1), weights.repeat(T // 400, 1)
    assert torch.equal(ops.mx_experts(many, many_index, many_weights, records, H, I)[-400:], want)


@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", [(9, 64, 32, 8, 3), (40, 100, 424, 20, 2),
                                                             (200, 256, 160, 8, 4), (300, 512, 256, 2, 2)])
def test_the_parts_in_turn(tokens, hidden, inner, experts, top_k):
    """dispatch, the products with bf16 rows, and combine."""
    h, packed, index, weights = _case(tokens, hidden, inner, experts, top_k)
    records = ops.mx_quantize_experts(packed, hidden, inner)
    plan = ops.dispatch(index, experts)
    rows = torch.empty((tokens * top_k, hidden), dtype=torch.bfloat16, device=DEV)
    ops.mx_grouped_swiglu(h, plan, weights.view(-1), records, hidden, inner, rows)
    got = ops.combine(rows, index, plan, hidden, accumulate_fp32=True)
    _check(got, h, index, weights, packed, hidden, inner, rows=torch.bfloat16)


@pytest.mark.parametrize("tokens", [40, 300])
@pytest.mark.parametrize("power", [90, -100])
def test_outputs_of_any_size(tokens, power):
    """A power of two in the last weight is one in the outputs."""
    H, I, E, K = 100, 64, 4, 2
    h, packed, index, weights = _case(tokens, H, I, E, K)
    want = ops.mx_experts(h, index, weights, ops.mx_quantize_experts(packed, H, I), H, I)
    packed[:, 2 * H * I:] *= 2.0 ** power
    got = ops.mx_experts(h, index, weights, ops.mx_quantize_experts(packed, H, I), H, I)
    assert torch.equal(got.double(), want.double() * 2.0 ** power)


@pytest.mark.parametrize("tokens", [40, 300])
def test_a_column_that_is_not_finite_stays_alone(tokens):
    H, I, E, K = 96, 64, 4, 2
    h, packed, index, weights = _case(tokens, H, I, E, K)
    want = ops.mx_experts(h, index, weights, ops.mx_quantize_experts(packed, H, I), H, I)
    packed[2, 2 * H * I + 37 * I + 5] = float("inf")       # of expert 2's down, output 37
    got = ops.mx_experts(h, index, weights, ops.mx_quantize_experts(packed, H, I), H, I)
    bad = torch.zeros((tokens, H), dtype=torch.bool, device=DEV)
    bad[(index == 2).any(1), 37] = True
    assert bad.any() and torch.equal(torch.isnan(got), bad)
    assert torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("tokens", [3, 40, 300])
def test_a_route_weight_that_is_not_finite_stays_in_its_token(tokens):
    H, I, E, K = 96, 64, 4, 2
    h, packed, index, weights = _case(tokens, H, I, E, K)
    records = ops.mx_quantize_experts(packed, H, I)
    want = ops.mx_experts(h, index, weights, records, H, I)
    weights[1, 0], weights[2, 1] = float("inf"), float("nan")
    got = ops.mx_experts(h, index, weights, records, H, I)
    assert not torch.isfinite(got[1:3]).any()
    there = [t for t in range(tokens) if t not in (1, 2)]
    assert torch.equal(got[there], want[there])


def test_two_calls_at_once():
    """Each call has scratch memory of its own."""
    H, I, E, K = 512, 256, 16, 4
    cases = [_case(t, H, I, E, K, seed=t) for t in (1, 300)]
    records = [ops.mx_quantize_experts(c[1], H, I) for c in cases]
    want = [ops.mx_experts(c[0], c[2], c[3], r, H, I) for c, r in zip(cases, records)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, (c, r) in enumerate(zip(cases, records)):
            got[i].append(ops.mx_experts(c[0], c[2], c[3], r, H, I, stream=streams[i]))
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(o, w) for o in outs)


@torch.inference_mode()
def test_a_model_with_mx_experts_prompt_and_decoding():
    """Every layer's experts in a model's own forwards, a prompt and single
    tokens after it, against the reference on what the layer was given."""
    from transformers import Qwen3MoeConfig, Qwen3MoeForCausalLM

    from specfit_amd.runtime import install_hip_attention, install_hip_norms, install_mx_experts

    torch.manual_seed(3)
    config = Qwen3MoeConfig(vocab_size=96, hidden_size=64, intermediate_size=48, moe_intermediate_size=32,
                            num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                            num_experts=6, num_experts_per_tok=2, norm_topk_prob=True)
    model = Qwen3MoeForCausalLM(config).to(torch.bfloat16).eval().to(DEV)
    packed = {}
    for i, layer in enumerate(model.model.layers):
        experts = layer.mlp.experts
        for p in experts.parameters():
            p.normal_(0, 0.2)
        packed[i] = torch.cat([experts.gate_up_proj.flatten(1), experts.down_proj.flatten(1)], 1)
    assert install_mx_experts(model) == 2 and install_mx_experts(model) == 0
    install_hip_norms(model), install_hip_attention(model)
    seen = []
    for i, layer in enumerate(model.model.layers):
        assert isinstance(layer.mlp.experts, Qwen3MXExperts)
        layer.mlp.experts.register_forward_hook(lambda m, a, o, i=i: seen.append((i, *a, o)))
    ids = torch.randint(0, 96, (1, 300), device=DEV)
    out = model(input_ids=ids, use_cache=True)
    for _ in range(3):
        assert torch.isfinite(out.logits).all()
        out = model(input_ids=out.logits[:, -1:].argmax(-1), past_key_values=out.past_key_values, use_cache=True)
    assert len(seen) == 8 and {s[1].shape[0] for s in seen} == {300, 1}
    for i, hidden, index, weights, got in seen:
        _check(got, hidden, index, weights.to(torch.bfloat16), packed[i], 64, 32)


def _even(tokens, experts, top_k):
    """Routes in turn: as many rows for one expert as for another."""
    t = torch.arange(tokens, device=DEV)[:, None]
    return (t * top_k + torch.arange(top_k, device=DEV)) % experts


# Two routes a token: without a dispatch; then 5 rows an expert (wavefronts), 20, 50,
# 100 and 150 (tiles of 32, 64 and 128 rows, and of 128 with one of 32).
FORMS = [(3, 4), (100, 40), (100, 10), (100, 4), (200, 4), (300, 4)]


@pytest.mark.parametrize("tokens,experts", FORMS)
def test_zeros_stay_zeros_under_large_route_weights(tokens, experts):
    """A token of zeros and outputs that no weight reaches are 0 whatever finite
    weight their routes have, and the others what they are."""
    H, I, K = 160, 64, 2
    h, packed, _, weights = _case(tokens, H, I, experts, K)
    index = _even(tokens, experts, K)
    packed.view(experts, 3, -1)[:, 2].view(experts, H, I)[:, 32:64] = 0
    sizes = torch.tensor([3.984375, 4.0, -8.0, 100.0, -2.0 ** 40], device=DEV, dtype=torch.bfloat16)
    weights = sizes[torch.arange(tokens * K, device=DEV) % 5].view(tokens, K).clone()
    empty = [1, tokens // 2, tokens - 1]
    h[empty] = 0
    weights[1] = torch.tensor([3e38, -3e38], device=DEV)
    records = ops.mx_quantize_experts(packed, H, I)
    got = ops.mx_experts(h, index, weights, records, H, I)
    assert torch.isfinite(got).all()
    assert not got[empty].any() and not got[:, 32:64].any()
    want, slack = ref.experts(h, index, weights, packed, H, I)
    assert (got.double() - want).abs().le(slack).all()
    rows = torch.full((tokens * K, H), 7.0, dtype=torch.bfloat16, device=DEV)
    plan = ops.dispatch(index, experts)
    ops.mx_grouped_swiglu(h, plan, weights.view(-1), records, H, I, rows)
    assert not rows[:, 32:64].any()
    token = plan.perm_pos.long() // K
    assert not rows[torch.isin(token, torch.tensor(empty, device=DEV))].any()


@pytest.mark.parametrize("tokens,experts", FORMS)
def test_tiny_sums_under_large_route_weights(tokens, experts):
    """Sums near 2^-116 and weights of 2^30: neither has to be taken past fp32's
    range on the way to their product."""
    H, I, K = 160, 64, 2
    h, packed, _, weights = _case(tokens, H, I, experts, K)
    index, weights = _even(tokens, experts, K), weights * 2.0 ** 30
    packed[:, 2 * H * I:] *= 2.0 ** -116
    got = ops.mx_experts(h, index, weights, ops.mx_quantize_experts(packed, H, I), H, I)
    want, slack = ref.experts(h, index, weights, packed, H, I)
    # A sum's terms and parts below 2^-126 may count as 0: 64 terms of a route, K routes.
    slack = slack + I * 2.0 ** -126 * weights.double().abs().sum(1, keepdim=True)
    assert (got.double() - want).abs().le(slack).all()


def _moe_model(layers=3):
    from transformers import Qwen3MoeConfig, Qwen3MoeForCausalLM

    torch.manual_seed(5)
    config = Qwen3MoeConfig(vocab_size=64, hidden_size=64, intermediate_size=48, moe_intermediate_size=32,
                            num_hidden_layers=layers, num_attention_heads=2, num_key_value_heads=1, head_dim=32,
                            num_experts=4, num_experts_per_tok=2)
    return Qwen3MoeForCausalLM(config).to(torch.bfloat16).eval().to(DEV)


def test_a_model_that_is_refused_stays_as_it_was():
    from specfit_amd.runtime import install_mx_experts

    model = _moe_model()
    before = [layer.mlp.experts for layer in model.model.layers]
    last = before[-1]
    good = last.act_fn
    last.act_fn = torch.nn.GELU()
    with pytest.raises(ValueError, match="silu"):
        install_mx_experts(model)
    last.act_fn = good
    last.to("cpu")
    with pytest.raises(ValueError, match="device"):
        install_mx_experts(model)
    last.to(DEV)
    kept, last.gate_up_proj = last.gate_up_proj, torch.nn.Parameter(last.gate_up_proj[:, 2:].contiguous())
    with pytest.raises(ValueError, match="intermediate"):
        install_mx_experts(model)
    last.gate_up_proj = kept
    assert all(layer.mlp.experts is b for layer, b in zip(model.model.layers, before))
    with pytest.raises(ValueError, match="from_module"):
        install_mx_experts(last)
    assert "" not in last._modules
    assert install_mx_experts(model) == 3
    assert all(isinstance(layer.mlp.experts, Qwen3MXExperts) for layer in model.model.layers)


def test_layers_are_released_one_by_one(monkeypatch):
    import gc
    import weakref

    from specfit_amd.runtime import install_mx_experts

    model = _moe_model()
    old = [weakref.ref(layer.mlp.experts.gate_up_proj) for layer in model.model.layers]
    make, alive = Qwen3MXExperts.from_module.__func__, []

    def from_module(cls, experts):
        gc.collect()
        alive.append([r() is not None for r in old])
        return make(cls, experts)

    monkeypatch.setattr(Qwen3MXExperts, "from_module", classmethod(from_module))
    assert install_mx_experts(model) == 3
    assert alive == [[True, True, True], [False, True, True], [False, False, True]]


def test_layers_that_share_their_experts():
    from specfit_amd.runtime import install_mx_experts

    model = _moe_model()
    layers = model.model.layers
    layers[2].mlp.experts = layers[0].mlp.experts
    assert install_mx_experts(model) == 2
    assert layers[2].mlp.experts is layers[0].mlp.experts and isinstance(layers[0].mlp.experts, Qwen3MXExperts)
    assert isinstance(layers[1].mlp.experts, Qwen3MXExperts)


@pytest.mark.parametrize("tokens", [3, 200])
def test_one_experts_records_may_have_any_stride(tokens):
    H, I = 64, 32
    h, packed, index, weights = _case(tokens, H, I, 1, 1)
    records = ops.mx_quantize_experts(packed, H, I)
    other = records.as_strided(records.shape, (1, 1))
    assert other.stride() == (1, 1) and other.is_contiguous()
    assert torch.equal(ops.mx_experts(h, index, weights, other, H, I), ops.mx_experts(h, index, weights, records, H, I))
    assert torch.equal(ops.mx_routed_swiglu(h, index, weights, other, H, I),
                       ops.mx_routed_swiglu(h, index, weights, records, H, I))
    plan, rows = ops.dispatch(index, 1), torch.empty((2, tokens, H), dtype=torch.bfloat16, device=DEV)
    for r, out in zip((other, records), rows):
        ops.mx_grouped_swiglu(h, plan, weights.view(-1), r, H, I, out)
    assert torch.equal(rows[0], rows[1])


def _integers(experts, H, I, low_bits, powers):
    """Experts in pairs (2p, 2p + 1) whose outputs for a token that holds 1 in its
    first place are whole numbers of 11 bits, apart in the last ``low_bits`` of them,
    times ``powers`` [H].  Gates are 32, where silu is the identity in fp32; the
    activations are 1, 2, ... 1,024, the numbers' bits lie in down: every product and
    sum is exact."""
    g = torch.Generator(device=DEV).manual_seed(experts)
    first = torch.randint(1024, 2048, (experts // 2, H), generator=g, device=DEV)
    other = first ^ torch.randint(0, 1 << low_bits, first.shape, generator=g, device=DEV)
    numbers = torch.stack([first, other], 1).flatten(0, 1)
    gate, up = (torch.zeros((experts, I, H), device=DEV) for _ in range(2))
    down = torch.zeros((experts, H, I), device=DEV)
    gate[:, :, 0] = 32
    bit = torch.arange(11, device=DEV)
    up[:, :11, 0] = torch.exp2(bit - 5.0)
    down[:, :, :11] = (numbers[..., None] >> bit & 1) * powers[:, None]
    return numbers, torch.cat([w.flatten(1) for w in (gate, up, down)], 1).to(torch.bfloat16)


@pytest.mark.parametrize("tokens,experts", FORMS)
@pytest.mark.parametrize("H", [64, 100, 328])
def test_routes_keep_eleven_bits_until_they_are_added(H, tokens, experts):
    """The difference of two routes of 11 bits, some of them 2^-24 of the others of
    their 32 columns: one bit less in a route's row, or an exponent that is off, would
    show."""
    I, K = 64, 2
    powers = torch.where(torch.arange(H, device=DEV) % 3 == 1, 2.0 ** -24, 1.0)
    numbers, packed = _integers(experts, H, I, 7, powers)
    h = torch.zeros((tokens, H), dtype=torch.bfloat16, device=DEV)
    h[:, 0] = 1
    pair = torch.arange(tokens, device=DEV) % (experts // 2)
    index = torch.stack([2 * pair, 2 * pair + 1], 1)
    weights = torch.tensor([1.0, -1.0], device=DEV, dtype=torch.bfloat16).expand(tokens, K).contiguous()
    got = ops.mx_experts(h, index, weights, ops.mx_quantize_experts(packed, H, I), H, I)
    want = (numbers[2 * pair] - numbers[2 * pair + 1]) * powers
    assert torch.equal(got.float(), want)


@pytest.mark.parametrize("H,I", [(256, 128), (96, 424)])
def test_chunks_of_every_height_in_one_launch(H, I):
    """Experts with as many rows as make full chunks, tall rests, which come first,
    and the rests of 64 and of 32 rows behind them."""
    counts = [0, 1, 20, 33, 64, 100, 128, 129, 300, 0, 32, 65]
    tokens = sum(counts)
    assert tokens > 16 * len(counts)      # both products by tiles of up to 128 rows
    rests = [c % 128 for c in counts if c % 128]
    assert any(c >= 128 for c in counts) and any(r > 64 for r in rests) \
        and any(32 < r <= 64 for r in rests) and any(r <= 32 for r in rests)
    h, packed, _, weights = _case(tokens, H, I, len(counts), 1)
    index = torch.repeat_interleave(torch.arange(len(counts), device=DEV), torch.tensor(counts, device=DEV))
    index = index[torch.randperm(tokens, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)][:, None]
    weights = torch.rand((tokens, 1), generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).to(torch.bfloat16)
    records = ops.mx_quantize_experts(packed, H, I)
    got = ops.mx_experts(h, index, weights, records, H, I)
    _check(got, h, index, weights, packed, H, I)
    # An expert's rows by themselves, in chunks of their own: the same sums.
    for e in (2, 6, 8):
        mine = index[:, 0] == e
        rows = torch.empty((int(mine.sum()), H), dtype=torch.bfloat16, device=DEV)
        ops.mx_grouped_swiglu(h[mine], ops.dispatch(torch.zeros_like(index[mine]), 1), weights[mine].view(-1),
                              records[e:e + 1], H, I, rows)
        # Both round the same fp32 row to bf16, one by way of 11 bits: a step of bf16, and
        # what a block of 11 bits loses below 2^-28 of its largest.
        alone, among = rows.float(), got[mine].float()
        step = 2.0 ** -7 * among.abs() + 2.0 ** -38 * among.abs().amax(1, keepdim=True)
        assert (alone - among).abs().le(step).all()


@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", [(1, 1, 1, 1, 1), (200, 1, 1, 2, 1), (300, 5, 3, 3, 2),
                                                             (30, 64, 32, 40, 32), (150, 64, 32, 64, 12),
                                                             (9, 7, 33, 256, 32)])
def test_smallest_sizes_and_many_routes(tokens, hidden, inner, experts, top_k):
    h, packed, index, weights = _case(tokens, hidden, inner, experts, top_k)
    want, slack = ref.experts(h, index, weights, packed, hidden, inner)
    got = ops.mx_experts(h, index, weights, ops.mx_quantize_experts(packed, hidden, inner), hidden, inner)
    assert (got.double() - want).abs().le(slack).all()


@pytest.mark.parametrize("tokens", [1, 20, 300])
def test_far_experts(tokens):
    """Records past 32 bits of offset."""
    H, I, E = 4096, 4096, 180
    h, packed, index, weights = _case(tokens, H, I, 2, 1)
    near = ops.mx_quantize_experts(packed, H, I)
    assert (E - 2) * near.shape[1] > 1 << 32
    far = torch.zeros((E, near.shape[1]), dtype=torch.uint8, device=DEV)
    far[-2:] = near
    pad = torch.arange(E - 2, device=DEV)[:, None]       # so that as many rows fall to an expert, in either form
    index = torch.cat([index, pad % 2]) if tokens > 1 else index
    h, weights = (torch.cat([t, t[:1].expand(index.shape[0] - tokens, -1)]) for t in (h, weights))
    out = [torch.empty((index.shape[0], H), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    table = torch.tensor([E - 2, E - 1], dtype=torch.int32, device=DEV)
    plan = ops.dispatch(index, 2)
    ops.mx_grouped_swiglu(h, plan, weights.view(-1), near, H, I, out[0])
    ops.mx_grouped_swiglu(h, plan, weights.view(-1), far, H, I, out[1], slot_of_expert=table)
    assert torch.equal(out[0], out[1])
    assert torch.equal(ops.mx_routed_swiglu(h[:2], index[:2], weights[:2], near, H, I),
                       ops.mx_routed_swiglu(h[:2], index[:2] + E - 2, weights[:2], far, H, I))


@pytest.mark.parametrize("tokens,experts", FORMS)
def test_absent_experts_and_bad_tokens_in_every_form(tokens, experts):
    """Routes to experts that the layer does not have count for nothing, alone and
    beside others; a token that is not finite spoils itself only."""
    H, I, K = 96, 64, 2
    h, packed, _, weights = _case(tokens, H, I, experts, K)
    index = _even(tokens, experts, K)
    records = ops.mx_quantize_experts(packed, H, I)
    index[0, 1], index[1] = experts, torch.tensor([-1, 2 ** 40], device=DEV)
    if tokens > 64:
        index[tokens // 2:tokens // 2 + 30] = -5
    got = ops.mx_experts(h, index, weights, records, H, I)
    _check(got, h, index, weights, packed, H, I)
    absent = ((index < 0) | (index >= experts)).all(1)
    assert absent.any() and not got[absent].any()
    h[2, 40], h[tokens - 1, 0], h[1, 7] = float("inf"), float("nan"), float("nan")
    bad = torch.zeros(tokens, dtype=torch.bool, device=DEV)
    bad[2] = bad[tokens - 1] = True          # token 1 has no expert to read it
    again = ops.mx_experts(h, index, weights, records, H, I)
    assert torch.isnan(again[bad]).all() and torch.equal(again[~bad], got[~bad])
    index[:] = -1
    assert not ops.mx_experts(h, index, weights, records, H, I).any()
