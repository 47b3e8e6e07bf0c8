"""Each kernel of the block attention (K10) against the plain 64-bit form: the
direct and the staged one, unsplit and with both ways of merging splits.  Bounds
count the kernels' roundings (see _block_reference.attention)."""
import math

import pytest
import torch

from _block_forms import CASES, ONE_OF_EACH, form_of, splits_of
from _block_reference import attention, held_rows
from specfit_amd import ops
from specfit_amd.runtime import BlockKVCache

pytestmark = pytest.mark.gpu

EACH = list(ONE_OF_EACH.values())
ALL = CASES + [c for c in EACH if c not in CASES]
SPLIT = [c for c in ALL if splits_of(c) > 1]


def _name(case):
    return "x".join(map(str, case))


def _rand(g, *shape):
    return torch.randn(shape, generator=g).to(torch.bfloat16)


def _inputs(case, g):
    B, Hq, H, D, Q, S = case
    return _rand(g, B, Hq, Q, D), _rand(g, B, H, S, D), _rand(g, B, H, S, D)


def _cache(device, case, k, v, held, folded, tail=None):
    """The sequences with ``folded`` blocks in 8 bits, in appends of at most
    ``tail`` tokens (a ring that goes round) or at once."""
    B, _, H, D, _, S = case
    cache = BlockKVCache(1, H, D, S, batch=B, held=held, tail_tokens=tail or S, device=device)
    step = tail or max(1, folded * 64)
    for at in range(0, folded * 64, step):
        end = min(at + step, folded * 64)
        cache.append(0, k[:, :, at:end].to(device), v[:, :, at:end].to(device))
        cache.commit()
    cache.append(0, k[:, :, folded * 64:].to(device), v[:, :, folded * 64:].to(device))
    assert cache.blocks.folded == folded
    return cache


def _mask(kind, g, case):
    B, _, _, _, Q, S = case
    if kind == "causal":
        return None
    if kind == "tree":  # over the new keys alone: chains with side branches
        m = torch.eye(Q, dtype=torch.bool)
        for i in range(1, Q):
            m[i] |= m[int(torch.randint(max(0, i - 9), i, (1,), generator=g))]
        return m.view(1, 1, Q, Q)
    if kind == "padded":
        pad = torch.randint(0, S - Q + 1, (B,), generator=g)
        pad[-1] = S  # nothing but padding
        at = torch.arange(S)
        causal = at[None] <= S - Q + torch.arange(Q)[:, None]
        return (causal[None] & (at >= pad[:, None, None])).view(B, 1, Q, S)
    m = torch.rand((B, 1, Q, max(1, S - 11)), generator=g) < 0.2
    m[:, :, ::4] = False
    return m


def _check(out, q, k, v, mask, scale):
    want, bound = attention(q, k, v, mask, scale)
    worst = ((out.cpu().double() - want).abs() / bound).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("kind,held,part", [
    ("causal", "e4m3", "all"), ("causal", "int8", "none"), ("tree", "int8", "all"),
    ("tree", "e4m3", "half"), ("padded", "e4m3", "all"), ("rows", "int8", "half")])
@pytest.mark.parametrize("case", ALL, ids=_name)
def test_forms(device, case, kind, held, part):
    """``part``: of the complete blocks before the last tokens, in 8 bits."""
    B, Hq, H, D, Q, S = case
    g = torch.Generator().manual_seed(Q + S)
    q, k, v = _inputs(case, g)
    folded = {"none": 0, "half": (S // 64) // 2, "all": (S - 1) // 64}[part]
    cache = _cache(device, case, k, v, held, folded, tail=None if part == "none" else max(S - folded * 64, 500))
    mask = _mask(kind, g, case)
    scale = D ** -0.5
    out = cache.attend(0, q.to(device), None if mask is None else mask.to(device), scale)
    # The reference takes its time: two heads of each of two sequences, and the first
    # KV head and the last.
    for b in {0, B - 1}:
        for h in {0, Hq - 1}:
            kv = h // (Hq // H)
            kk, vv = (held_rows(t[b:b + 1, kv:kv + 1], folded, held) for t in (k, v))
            m = mask if mask is None or mask.shape[0] == 1 else mask[b:b + 1]
            _check(out[b:b + 1, :, h:h + 1], q[b:b + 1, h:h + 1], kk, vv, m, scale)
    if kind == "padded":
        assert not out[-1].any()
    # The other heads: against those of a call in which they change places.
    turned = cache.attend(0, q.view(B, H, Hq // H, Q, D).flip(2).reshape(q.shape).to(device),
                          None if mask is None else mask.to(device), scale)
    back = turned.view(B, Q, H, Hq // H, D).flip(3).reshape(out.shape)
    assert torch.equal(back, out)


@pytest.mark.parametrize("held", ("e4m3", "int8"))
@pytest.mark.parametrize("case", EACH, ids=_name)
def test_values_that_are_not_finite(device, case, held):
    """In a folded block, in the last block and in the first: NaN where the codes hold
    them, as they are in bf16; only in the element and the rows that admit the key."""
    B, Hq, H, D, Q, S = case
    g = torch.Generator().manual_seed(Q)
    q, k, v = _inputs(case, g)
    folded = (S - 1) // 64
    mask = torch.rand((1, 1, Q, S), generator=g) < 0.7
    for place, value in ((0, math.inf), (S - 1, math.inf), (S - 1, -math.inf), (S // 2, math.nan)):
        mask[..., place] = torch.arange(Q) % 2 == 0
        v[-1, -1, place, 7] = 0.0
        clean = _cache(device, case, k, v, held, folded).attend(0, q.to(device), mask.to(device)).cpu()
        bad = v.clone()
        bad[-1, -1, place, 7] = value
        out = _cache(device, case, k, bad, held, folded).attend(0, q.to(device), mask.to(device)).cpu()
        seen = out[-1, ::2, Hq - Hq // H:, 7]
        if place // 64 < folded or math.isnan(value):
            assert bool(seen.isnan().all())
        else:
            assert bool((seen.isnan() | (seen == value)).all()) and not seen.isfinite().any()
        out[-1, ::2, Hq - Hq // H:, 7] = clean[-1, ::2, Hq - Hq // H:, 7]
        assert torch.equal(out, clean)


@pytest.mark.parametrize("scale", (0.0, -0.3, 40.0))
@pytest.mark.parametrize("case", EACH, ids=_name)
def test_scales_of_the_scores(device, case, scale):
    B, Hq, H, D, Q, S = case
    g = torch.Generator().manual_seed(S)
    q, k, v = _inputs(case, g)
    folded = (S - 1) // 64
    out = _cache(device, case, k, v, "int8", folded).attend(0, q.to(device), None, scale)
    kk, vv = (held_rows(t[-1:, -1:], folded, "int8") for t in (k, v))
    _check(out[-1:, :, -1:], q[-1:, -1:], kk, vv, None, scale)


@pytest.mark.parametrize("case", EACH, ids=_name)
def test_blocks_of_very_different_scales(device, case):
    """Value scales change from block to block by up to 2^40, key scales by 2^10."""
    B, Hq, H, D, Q, S = case
    g = torch.Generator().manual_seed(D)
    q, k, v = _inputs(case, g)
    block = torch.arange(S) // 64
    v = (v * torch.exp2(torch.tensor([0., 20, -20, 3, -3, 10, -40, 0, 1])[block % 9])[:, None]).bfloat16()
    k = (k * torch.exp2(torch.tensor([0., -5, 2, -8, 1, 0, 0, 2])[block % 8])[:, None]).bfloat16()
    folded = (S - 1) // 64
    for held in ("e4m3", "int8"):
        out = _cache(device, case, k, v, held, folded).attend(0, q.to(device), None, 0.125)
        kk, vv = (held_rows(t[:1, :1], folded, held) for t in (k, v))
        _check(out[:1, :, :1], q[:1, :1], kk, vv, None, 0.125)


@pytest.mark.parametrize("kind", ("tokens first", "odd offset", "strided"))
@pytest.mark.parametrize("case", ((5, 32, 4, 128, 130, 260), (5, 16, 4, 128, 333, 833)), ids=_name)
def test_layouts(device, case, kind):
    B, Hq, H, D, Q, S = case
    g = torch.Generator().manual_seed(9)
    q, k, v = _inputs(case, g)
    cache = _cache(device, case, k, v, "e4m3", (S - 1) // 64)
    if kind == "tokens first":
        mine = q.transpose(1, 2).contiguous().to(device).transpose(1, 2)
    elif kind == "odd offset":
        mine = torch.cat([q[..., :1], q], -1).to(device)[..., 1:]
    else:
        mine = q.repeat_interleave(2, -1).to(device)[..., ::2]
    wide = torch.rand((B, 1, Q, S + 5), generator=g) < 0.7
    for mask in (wide[..., 5:], wide[..., 2:40], wide[..., :0],
                 wide.transpose(2, 3).contiguous().transpose(2, 3)[..., :S]):
        whole = torch.ones((B, 1, Q, S), dtype=torch.bool)
        whole[..., S - mask.shape[-1]:] = mask
        got = cache.attend(0, mine, mask.to(device))
        assert torch.equal(got, cache.attend(0, q.to(device), whole.to(device)))


@pytest.mark.parametrize("case", SPLIT, ids=_name)
def test_without_room_for_scratch(device, case, monkeypatch):
    """The same keys in one piece: the result moves by roundings only."""
    B, Hq, H, D, Q, S = case
    g = torch.Generator().manual_seed(8)
    q, k, v = _inputs(case, g)
    folded = (S - 1) // 64
    cache = _cache(device, case, k, v, "int8", folded)
    monkeypatch.setattr(ops, "_block_attention_workspace", lambda *a: 0)
    out = cache.attend(0, q.to(device))
    kk, vv = (held_rows(t[-1:, -1:], folded, "int8") for t in (k, v))
    _check(out[-1:, :, -1:], q[-1:, -1:], kk, vv, None, D ** -0.5)


@pytest.mark.parametrize("case", EACH, ids=_name)
def test_captured_repeated_and_on_two_streams(device, case):
    B, Hq, H, D, Q, S = case
    g = torch.Generator().manual_seed(12)
    q, k, v = _inputs(case, g)
    cache = _cache(device, case, k, v, "int8", (S - 1) // 64)
    q = q.to(device)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        cache.attend(0, q)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = cache.attend(0, q)
    other = _rand(g, *q.shape).to(device)
    for turn in range(4):
        q.copy_(_rand(g, *q.shape).to(device))
        graph.replay()
        got = captured.clone()
        torch.cuda.synchronize()
        want = cache.attend(0, q)
        assert torch.equal(got, want), turn
    want = [cache.attend(0, q), cache.attend(0, other)]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(cache.attend(0, (q, other)[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(o, want[i]) for o in outs[i])


@pytest.mark.parametrize("case", EACH, ids=_name)
def test_a_row_keeps_its_bits_beside_very_large_scores(device, case):
    """Scores of other rows, up to 2^40 and infinite, change nothing in a row."""
    B, Hq, H, D, Q, S = case
    g = torch.Generator().manual_seed(5)
    q, k, v = _inputs(case, g)
    q = q * 4  # peaked: a last bit of a score shows
    cache = _cache(device, case, k, v, "e4m3", (S - 1) // 64)
    clean = cache.attend(0, q.to(device)).cpu()
    loud = torch.rand((B, Hq, Q), generator=g) < 0.15
    loud[:, 0, 0] = True
    for size in (2.0 ** 40, math.inf):
        p = torch.where(loud[..., None], (q.float() * size).bfloat16(), q)
        out = cache.attend(0, p.to(device)).cpu()
        keep = ~loud.transpose(1, 2)
        assert torch.equal(out[keep], clean[keep])


@pytest.mark.parametrize("held", ("e4m3", "int8"))
@pytest.mark.parametrize("case", [c for c in ((1, 8, 2, 64, 1, 3), (4, 8, 2, 128, 1, 9),
                                              (2, 16, 4, 128, 5, 20), (2, 8, 4, 64, 30, 70),
                                              (2, 64, 4, 128, 9, 300)) if form_of(c)[0] == 16],
                         ids=_name)
def test_weights_of_the_direct_form(device, case, held):
    """Kept to 2^-16 of themselves (two bf16 terms of half steps 2^-8 each), where one
    term would lose 2^-8; beside it S sums of up to a step, 2^-23, of the values' sizes."""
    B, Hq, H, D, Q, S = case
    g = torch.Generator().manual_seed(S)
    q, k, v = _inputs(case, g)
    folded = (S - 1) // 64
    scale = D ** -0.5
    out = _cache(device, case, k, v, held, folded).attend(0, q.to(device), None, scale)
    kk, vv = (held_rows(t, folded, held) for t in (k, v))
    want, bound = attention(q, kk, vv, None, scale)
    size, _ = attention(q, kk, vv.abs(), None, scale)
    bound = bound - (2.0 ** -8 - 2.0 ** -16 - S * 2.0 ** -23) * size
    worst = ((out.cpu().double() - want).abs() / bound).max().item()
    assert worst <= 1.0, worst
