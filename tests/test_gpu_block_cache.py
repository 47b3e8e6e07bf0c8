"""The block cache and its attention (K9, K10) against plain 64-bit forms.

What the cache gives back and its scales are exact; the attention is held to
a bound that counts its roundings (see _block_reference.attention)."""
import math

import pytest
import torch

from _block_reference import BLOCK, attention, fold, held_rows
from specfit_amd import ops
from specfit_amd.runtime import BlockKVCache

pytestmark = pytest.mark.gpu
HELD = ("e4m3", "int8")


def _rand(g, *shape, std=1.0):
    return (torch.randn(shape, generator=g) * std).to(torch.bfloat16)


def _cache(device, *, H=2, D=64, capacity=512, batch=1, layers=1, held="e4m3", tail=4096):
    return BlockKVCache(layers, H, D, capacity, batch=batch, held=held, tail_tokens=tail,
                        device=device)


def _same(a, b):
    """Equal values, NaN where NaN."""
    a, b = a.cpu().double(), b.cpu().double()
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def _check_attention(cache, q, k, v, mask, scale, held, *, layer=0):
    """cache holds k and v [B, H, S, D] (bf16, CPU)."""
    folded = cache.blocks.folded
    kk, vv = held_rows(k, folded, held), held_rows(v, folded, held)
    mine = cache.attend(layer, q.to(cache.blocks.device),
                        None if mask is None else mask.to(cache.blocks.device), scale)
    want, bound = attention(q, kk, vv, mask, scale)
    assert mine.dtype == torch.bfloat16 and mine.shape == want.shape
    err = (mine.cpu().double() - want).abs()
    worst = (err / bound).max().item()
    assert worst <= 1.0, worst
    return mine


# ------------------------------------------------------------------- fold --
@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("D", (64, 128))
def test_codes_and_scales_are_exact(device, held, D):
    """Blocks of every kind: ordinary, at a border of the scale, loud and
    quiet, zeros, subnormals, values that are not finite."""
    g = torch.Generator().manual_seed(D)
    blocks = [_rand(g, BLOCK, D), _rand(g, BLOCK, D, std=3e4), _rand(g, BLOCK, D, std=2.0 ** -50),
              _rand(g, BLOCK, D, std=2.0 ** -58), _rand(g, BLOCK, D, std=2.0 ** -70),
              torch.zeros(BLOCK, D).to(torch.bfloat16), _rand(g, BLOCK, D, std=2.0 ** 120),
              _rand(g, BLOCK, D, std=2.0 ** -130)]
    for top in (127.0, 128.0, 126.5, 448.0, 450.0, 446.0, 1.75, 1.7578125, 0.9921875, 1.0):
        b = _rand(g, BLOCK, D, std=top / 8).clamp(-top, top)
        b[5, 7] = -top
        blocks.append(b)
    ties = torch.arange(BLOCK * D).view(BLOCK, D) % 255 - 127  # halves between codes
    blocks.append((ties / 2).to(torch.bfloat16))
    tiny = (torch.arange(BLOCK * D).view(BLOCK, D) % 512).to(torch.bfloat16) * 2.0 ** -11
    tiny[0, 0] = 448.0  # e4m3's subnormals beside its largest value
    blocks.append(tiny.to(torch.bfloat16))
    for value in (math.nan, math.inf, -math.inf):
        b = _rand(g, BLOCK, D)
        b[3, 9], b[63, D - 1] = value, value
        blocks.append(b)
    blocks.append(torch.full((BLOCK, D), math.inf).to(torch.bfloat16))
    x = torch.stack(blocks)[None, None].expand(1, 2, -1, -1, -1).flatten(2, 3).contiguous()
    y = x.flip(2).contiguous()
    n = len(blocks)
    cache = _cache(device, D=D, capacity=n * BLOCK, held=held)
    cache.append(0, x.to(device), y.to(device))
    cache.commit()
    assert cache.folded_tokens == n * BLOCK
    for t, got, scales in zip((x, y), cache.read(0), cache.scales(0)):
        want, scale = fold(t.unflatten(2, (n, BLOCK)), held)
        assert _same(scales, scale)
        assert _same(got, want.flatten(2, 3))


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("sizes", [(1,), (63, 1, 1), (64,), (65, 62, 3), (7, 120, 1, 1, 200), (300,)])
def test_appends_and_reads(device, held, D, sizes):
    """Any division of a sequence into appends gives the same cache; reads at
    any offsets."""
    g = torch.Generator().manual_seed(sum(sizes))
    S, B, H = sum(sizes), 2, 3
    k, v = _rand(g, B, H, S, D), _rand(g, B, H, S, D)
    cache = _cache(device, H=H, D=D, capacity=S, batch=B, held=held)
    at = 0
    for i, n in enumerate(sizes):
        cache.append(0, k[:, :, at:at + n].to(device), v[:, :, at:at + n].to(device))
        at += n
        if i % 2:
            cache.commit()
    folded = cache.blocks.folded
    for t, got in zip((k, v), cache.read(0)):
        assert _same(got, held_rows(t, folded, held))
    cache.commit()
    assert cache.folded_tokens == S // BLOCK * BLOCK
    want = [held_rows(t, S // BLOCK, held) for t in (k, v)]
    for start, stop in ((0, S), (S // 2, S), (S - 1, S), (S // 3, S // 3), (1, max(1, S - 1))):
        for w, got in zip(want, cache.read(0, start, stop)):
            assert _same(got, w[:, :, start:stop])


@pytest.mark.parametrize("kind", ("tokens first", "odd offset", "strided", "expanded"))
def test_layouts_of_appended_rows(device, kind):
    g = torch.Generator().manual_seed(5)
    B, H, T, D = 2, 2, 77, 64
    if kind == "tokens first":
        t = _rand(g, B, T, H, D).to(device).transpose(1, 2)
    elif kind == "odd offset":
        t = _rand(g, B, H, T, D + 3).to(device)[..., 3:]
    elif kind == "strided":
        t = _rand(g, B, H, T, 2 * D).to(device)[..., ::2]
    else:
        t = _rand(g, 1, 1, T, D).to(device).expand(B, H, T, D)
    cache = _cache(device, H=H, D=D, capacity=T, batch=B)
    cache.append(0, t, t)
    for got in cache.read(0):
        assert torch.equal(got, t)


@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("base,count,tree", [(0, 1, 1), (10, 3, 8), (60, 20, 61), (130, 100, 128),
                                             (5, 290, 400), (64, 0, 5), (7, 40, 40)])
def test_compaction(device, D, base, count, tree):
    """Accepted rows move to the front of the tree's, in every layer."""
    g = torch.Generator().manual_seed(base + count)
    layers, H = 3, 2
    keep = sorted(torch.randperm(tree, generator=g)[:count].tolist())
    ks = [_rand(g, 1, H, base + tree, D) for _ in range(layers)]
    vs = [_rand(g, 1, H, base + tree, D) for _ in range(layers)]
    cache = _cache(device, H=H, D=D, capacity=base + tree, layers=layers)
    for l in range(layers):
        cache.append(l, ks[l].to(device), vs[l].to(device))
    cache.compact(base, keep)
    rows = list(range(base)) + [base + p for p in keep]
    for l in range(layers):
        assert cache.get_seq_length(l) == len(rows)
        for t, got in zip((ks[l], vs[l]), cache.read(l)):
            assert _same(got, t[:, :, rows])
    cache.commit()
    for l in range(layers):
        for t, got in zip((ks[l], vs[l]), cache.read(l)):
            assert _same(got, held_rows(t[:, :, rows], len(rows) // BLOCK, "e4m3"))


@pytest.mark.parametrize("held", HELD)
def test_the_ring_goes_round(device, held):
    """A long sequence through a small tail: appends, rejected drafts,
    compactions and folds, block after block, with the attention at each step."""
    g = torch.Generator().manual_seed(17)
    H, D, capacity, tree = 2, 64, 700, 30
    cache = _cache(device, H=H, D=D, capacity=capacity, held=held, tail=tree)
    assert cache.blocks.ring_blocks == 2
    k, v = torch.empty(1, H, 0, D).bfloat16(), torch.empty(1, H, 0, D).bfloat16()
    step = 0
    while k.shape[2] + tree <= capacity:
        nk, nv = _rand(g, 1, H, tree, D), _rand(g, 1, H, tree, D)
        base = k.shape[2]
        cache.append(0, nk.to(device), nv.to(device))
        kept = sorted(torch.randperm(tree, generator=g)[:12].tolist())
        if step % 3 == 0:
            _check_attention(cache, _rand(g, 1, 4, tree, D), torch.cat([k, nk], 2),
                             torch.cat([v, nv], 2), None, 0.125, held)
        cache.compact(base, kept)
        k, v = torch.cat([k, nk[:, :, kept]], 2), torch.cat([v, nv[:, :, kept]], 2)
        cache.commit()
        step += 1
    assert cache.blocks.folded > 2 * cache.blocks.ring_blocks
    for t, got in zip((k, v), cache.read(0)):
        assert _same(got, held_rows(t, cache.blocks.folded, held))


# -------------------------------------------------------------- attention --
CASES = [  # batch, query heads, KV heads, D, prefix, new, mask
    (1, 4, 4, 64, 0, 1, None), (1, 8, 2, 128, 0, 65, None), (1, 32, 4, 128, 64, 1, None),
    (1, 32, 4, 128, 200, 1, None), (1, 14, 2, 64, 1000, 1, None), (1, 16, 1, 128, 4097, 1, None),
    (2, 12, 4, 128, 130, 7, None), (1, 32, 4, 128, 100, 61, "tree"), (1, 64, 4, 128, 700, 128, "tree"),
    (1, 40, 8, 128, 77, 33, "tree"), (3, 8, 2, 64, 150, 5, "padded"), (2, 4, 2, 128, 63, 130, "padded"),
    (1, 8, 2, 64, 300, 17, "rows"), (1, 32, 4, 128, 128, 300, None), (1, 4, 1, 64, 20000, 2, None),
    (1, 17, 1, 64, 190, 1, "tree"), (1, 5, 1, 128, 64, 64, None), (1, 16, 4, 128, 513, 200, None),
]


def _mask(kind, g, B, prefix, new):
    if kind is None:
        return None
    S = prefix + new
    if kind == "tree":  # over the new keys alone
        m = torch.eye(new, dtype=torch.bool)
        for i in range(1, new):
            m[i] |= m[int(torch.randint(max(0, i - 9), i, (1,), generator=g))]
        return m.view(1, 1, new, new)
    if kind == "padded":
        pad = torch.randint(0, prefix + 1, (B,), generator=g)
        pad[-1] = S  # nothing but padding
        at = torch.arange(S)
        causal = at[None] <= prefix + torch.arange(new)[:, None]
        return (causal[None] & (at >= pad[:, None, None])).view(B, 1, new, S)
    m = torch.rand((1, 1, new, S - 11), generator=g) < 0.2  # any pattern, rows of nothing among it
    m[:, :, ::4] = False
    return m


def _filled(device, g, B, H, D, prefix, new, held, *, std=1.0):
    k, v = _rand(g, B, H, prefix + new, D, std=std), _rand(g, B, H, prefix + new, D)
    cache = _cache(device, H=H, D=D, capacity=prefix + new, batch=B, held=held,
                   tail=max(prefix, new))
    if prefix:
        cache.append(0, k[:, :, :prefix].to(device), v[:, :, :prefix].to(device))
        cache.commit()
    cache.append(0, k[:, :, prefix:].to(device), v[:, :, prefix:].to(device))
    return cache, k, v


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("B,Hq,H,D,prefix,new,kind", CASES)
def test_attention(device, held, B, Hq, H, D, prefix, new, kind):
    g = torch.Generator().manual_seed(prefix + new)
    cache, k, v = _filled(device, g, B, H, D, prefix, new, held)
    mask = _mask(kind, g, B, prefix, new)
    out = _check_attention(cache, _rand(g, B, Hq, new, D), k, v, mask, D ** -0.5, held)
    if kind == "padded":
        assert not out[-1].any()
    if kind == "rows":
        # Row 0 of the mask admits none of its keys, but those before it.
        assert out[:, 0].any()


def test_rows_that_admit_nothing_are_zero(device):
    g = torch.Generator().manual_seed(1)
    for held, S, new in (("e4m3", 640, 3), ("int8", 64, 64), ("int8", 5, 5)):
        cache, k, v = _filled(device, g, 1, 2, 64, S - new, new, held)
        mask = torch.ones((1, 1, new, S), dtype=torch.bool)
        mask[:, :, 1] = False
        out = _check_attention(cache, _rand(g, 1, 4, new, 64), k, v, mask, 0.125, held)
        assert not out[:, 1].any() and out[:, 0].any()


def test_queries_more_than_keys(device):
    """Causal at the end: rows before the first key admit nothing."""
    g = torch.Generator().manual_seed(2)
    k = _rand(g, 1, 2, 9, 64)
    cache = _cache(device)
    cache.append(0, k.to(device), k.to(device))
    out = _check_attention(cache, _rand(g, 1, 4, 20, 64), k, k, None, 0.125, "e4m3")
    assert not out[:, :11].any()


def test_an_empty_cache_and_no_queries(device):
    cache = _cache(device)
    q = torch.ones((1, 4, 3, 64), dtype=torch.bfloat16, device=device)
    assert not cache.attend(0, q).any()
    assert cache.attend(0, q[:, :, :0]).shape == (1, 0, 4, 64)
    empty = torch.empty((1, 2, 0, 64), dtype=torch.bfloat16, device=device)
    cache.append(0, empty, empty)
    assert cache.get_seq_length() == 0
    assert cache.read(0)[0].shape == (1, 2, 0, 64)


@pytest.mark.parametrize("scale", (0.0, -0.3, 1e-4, 3.0, 40.0))
@pytest.mark.parametrize("rows", (1, 40))
def test_scales_of_the_scores(device, scale, rows):
    """A scale of 0 is the mean; negative and large ones keep their order."""
    g = torch.Generator().manual_seed(rows)
    cache, k, v = _filled(device, g, 1, 2, 64, 130, rows, "int8")
    _check_attention(cache, _rand(g, 1, 8, rows, 64), k, v, None, scale, "int8")


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("rows", (1, 40))
def test_blocks_of_very_different_scales(device, held, rows):
    """Value scales change from block to block by 2^40, key scales by 2^10."""
    g = torch.Generator().manual_seed(rows)
    S, D = 64 * 9 + rows, 64
    k, v = _rand(g, 1, 2, S, D), _rand(g, 1, 2, S, D)
    size = torch.exp2(torch.tensor([0, 20, -20, 3, -3, 10, -40, 0, 1, 0]).repeat_interleave(64)[:S].float())
    v = (v * size[:, None]).to(torch.bfloat16)
    k = (k * torch.exp2(torch.tensor([0, -5, 2, -8, 1, 0, 0, 2, -1, 0]).repeat_interleave(64)[:S].float())[:, None]).to(torch.bfloat16)
    cache = _cache(device, D=D, capacity=S, held=held)
    cache.append(0, k.to(device), v.to(device))
    cache.commit()
    _check_attention(cache, _rand(g, 1, 8, rows, D), k, v, None, 0.125, held)


def test_very_large_scores(device):
    """Scores near 2^30 in log2 units: the weight goes to the largest."""
    S, D = 200, 64
    k = torch.zeros(1, 1, S, D)
    k[0, 0, :, 0] = torch.arange(S) % 50
    k = k.to(torch.bfloat16)
    v = _rand(torch.Generator().manual_seed(3), 1, 1, S, D)
    cache = _cache(device, H=1, D=D, capacity=S, held="int8")
    cache.append(0, k.to(device), v.to(device))
    cache.commit()
    for rows in (1, 40):
        q = torch.zeros(1, 1, rows, D)
        q[..., 0] = 2.0 ** 24
        out = cache.attend(0, q.to(torch.bfloat16).to(device), torch.ones(
            (1, 1, rows, S), dtype=torch.bool, device=device), 1.0)
        # The keys that share the largest score (49): the mean of their values.
        want = held_rows(v, 3, "int8")[0, 0, [49, 99, 149, 199]].mean(0)
        err = (out[0, :, 0].cpu().double() - want).abs()
        assert bool((err <= 2.0 ** -7 * v[0, 0, [49, 99, 149, 199]].double().abs().mean(0) + 1e-6).all())


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("rows", (1, 9, 200))
@pytest.mark.parametrize("place", (10, 70, 200))  # two folded blocks, and the tail
def test_values_that_are_not_finite(device, held, rows, place):
    """An infinite or NaN value reaches the rows that admit its key, in its
    own element, and no others; what the cache keeps of it in 8 bits is NaN."""
    g = torch.Generator().manual_seed(rows)
    S, D, H, Hq = 210, 64, 2, 8
    k, v = _rand(g, 1, H, S, D), _rand(g, 1, H, S, D)
    q = _rand(g, 1, Hq, rows, D)
    mask = torch.ones((1, 1, rows, S), dtype=torch.bool)
    mask[:, :, ::2, place] = False

    def run(kk, vv):
        cache = _cache(device, H=H, D=D, capacity=S, held=held)
        cache.append(0, kk.to(device), vv.to(device))
        cache.commit()
        assert cache.blocks.folded == 3
        return cache.attend(0, q.to(device), mask.to(device), 0.125).cpu()

    zero = v.clone()
    zero[0, 1, place, 7] = 0.0
    clean = run(k, zero)
    for value in (math.inf, -math.inf, math.nan):
        bad = v.clone()
        bad[0, 1, place, 7] = value
        out = run(k, bad)
        seen = out[0, 1::2, Hq // 2:, 7]
        expect = math.nan if place < 192 else value
        assert bool((seen.isnan() if math.isnan(expect) else seen == expect).all())
        out[0, 1::2, Hq // 2:, 7] = clean[0, 1::2, Hq // 2:, 7]
        assert torch.equal(out, clean)
        # A key: the rows that admit it are NaN (or follow an infinite score).
        bad = k.clone()
        bad[0, 1, place, 7] = math.nan
        out = run(bad, v)
        assert bool(out[0, 1::2, Hq // 2:].isnan().all())
        assert bool(out[0, ::2].isfinite().all()) and bool(out[0, :, :Hq // 2].isfinite().all())


def test_infinities_of_both_signs(device):
    S, D = 100, 64
    g = torch.Generator().manual_seed(0)
    k, v = _rand(g, 1, 1, S, D), _rand(g, 1, 1, S, D)
    v[0, 0, 3, 5], v[0, 0, 90, 5], v[0, 0, 91, 6] = math.inf, -math.inf, -math.inf
    cache = _cache(device, H=1, D=D, capacity=S)
    cache.append(0, k.to(device), v.to(device))  # not committed: all in bf16
    out = cache.attend(0, _rand(g, 1, 2, 1, D).to(device))
    assert bool(out[..., 5].isnan().all()) and bool((out[..., 6] == -math.inf).all())
    assert bool(out[..., 7:].isfinite().all())


@pytest.mark.parametrize("rows", (1, 60))
def test_what_lies_behind_the_last_token_has_no_effect(device, rows):
    """Rejected drafts full of NaN stay in the ring; so do blocks of an
    earlier turn.  Nothing of them is seen, and their flags go when the blocks
    are written again."""
    g = torch.Generator().manual_seed(rows)
    D = 64
    k, v = _rand(g, 1, 2, 100 + rows, D), _rand(g, 1, 2, 100 + rows, D)
    q = _rand(g, 1, 4, rows, D)
    cache = _cache(device, D=D, capacity=600, tail=300)
    cache.append(0, k[:, :, :100].to(device), v[:, :, :100].to(device))
    junk = torch.full((1, 2, 150, D), math.nan).to(torch.bfloat16)
    cache.append(0, junk.to(device), junk.to(device))
    cache.crop(100)
    _check_attention(cache, q, k[:, :, :100], v[:, :, :100], None, 0.125, "e4m3")
    cache.append(0, k[:, :, 100:].to(device), v[:, :, 100:].to(device))
    _check_attention(cache, q, k, v, None, 0.125, "e4m3")
    cache.reset()
    cache.append(0, k.to(device), v.to(device))
    blocks = -(-(100 + rows) // BLOCK)
    assert not cache.blocks.tail_flags[0, :, :blocks].any()
    _check_attention(cache, q, k, v, None, 0.125, "e4m3")


def test_compaction_moves_flags(device):
    """An infinite value that is accepted keeps its effect in its new block."""
    g = torch.Generator().manual_seed(4)
    D = 64
    k, v = _rand(g, 1, 2, 130, D), _rand(g, 1, 2, 130, D)
    v[0, 0, 129, 3] = math.inf
    cache = _cache(device, D=D, capacity=130)
    cache.append(0, k.to(device), v.to(device))
    cache.compact(10, (0, 119))
    out = cache.attend(0, _rand(g, 1, 2, 1, D).to(device))
    assert bool((out[0, 0, 0, 3] == math.inf).all())
    mask = torch.ones((1, 1, 1, 12), dtype=torch.bool, device=device)
    mask[..., 11] = False
    assert bool(cache.attend(0, _rand(g, 1, 2, 1, D).to(device), mask).isfinite().all())


@pytest.mark.parametrize("kind", ("tokens first", "odd offset", "strided"))
def test_layouts_of_queries_and_masks(device, kind):
    g = torch.Generator().manual_seed(9)
    B, Hq, H, D, S, Q = 2, 4, 2, 64, 150, 6
    cache, k, v = _filled(device, g, B, H, D, S - Q, Q, "int8")
    if kind == "tokens first":
        q = _rand(g, B, Q, Hq, D).to(device).transpose(1, 2)
    elif kind == "odd offset":
        q = _rand(g, B, Hq, Q, D + 1).to(device)[..., 1:]
    else:
        q = _rand(g, B, Hq, Q, 2 * D).to(device)[..., ::2]
    wide = torch.rand((B, 1, Q, S + 5), generator=g) < 0.7
    for mask in (wide[..., 5:], wide[:1, ..., :S].expand(B, -1, -1, -1), wide[..., 2:40],
                 wide.transpose(2, 3).contiguous().transpose(2, 3)[..., :S], wide[..., :0]):
        _check_attention(cache, q, k, v, mask, 0.125, "int8")


def test_calls_without_room_for_scratch(device, monkeypatch):
    """With no workspace the keys are not split."""
    g = torch.Generator().manual_seed(8)
    cache, k, v = _filled(device, g, 1, 2, 64, 9000, 1, "int8")
    q = _rand(g, 1, 4, 1, 64)
    assert ops._block_attention_workspace(1, 1, 9001, 4, 2, 64) > 0
    monkeypatch.setattr(ops, "_block_attention_workspace", lambda *a: 0)
    _check_attention(cache, q, k, v, None, 0.125, "int8")


def test_captured_calls(device):
    """Two graphs that append and attend at their own lengths, replayed in turn
    with eager work between, against eager calls."""
    g = torch.Generator().manual_seed(12)
    H, D, S = 2, 64, 1500
    k, v = _rand(g, 1, H, S, D).to(device), _rand(g, 1, H, S, D).to(device)
    cache = _cache(device, H=H, D=D, capacity=S + 10, held="int8")
    cache.append(0, k, v)
    cache.commit()
    new = [[_rand(g, 1, H, n, D).to(device) for _ in range(2)] + [_rand(g, 1, 8, n, D).to(device)]
           for n in (1, 7)]

    def step(i):
        nk, nv, q = new[i]
        cache.append(0, nk, nv)
        out = cache.attend(0, q)
        cache.crop(S)
        return out

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for i in (0, 1):
            step(i)
    torch.cuda.current_stream().wait_stream(stream)
    graphs, outs = [], []
    for i in (0, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(i))
        graphs.append(graph)
    for turn in range(4):
        for i in (0, 1):
            for t in new[i]:
                t.copy_(_rand(g, *t.shape).to(device))
            graphs[i].replay()
            got = outs[i].clone()
            want = step(i)
            torch.cuda.synchronize()
            assert torch.equal(got, want), (turn, i)


def test_another_stream(device):
    g = torch.Generator().manual_seed(13)
    cache, k, v = _filled(device, g, 1, 2, 64, 1000, 3, "e4m3")
    q = _rand(g, 1, 4, 3, 64).to(device)
    want = cache.attend(0, q)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    got = ops.block_attention(cache.blocks, 0, q, 1003, None, 64 ** -0.5, stream=stream)
    stream.synchronize()
    assert torch.equal(got, want)


def test_another_stream_takes_its_own_copies(device):
    """Layouts that a call copies first: on the stream it was given, where the
    caller ordered the inputs, not behind what the current stream still does."""
    g = torch.Generator().manual_seed(16)
    key, value, q = (_rand(g, 1, h, n, 64) for h, n in ((2, 90), (2, 90), (4, 3)))
    swapped = lambda t: t.transpose(2, 3).contiguous().to(device).transpose(2, 3)  # noqa: E731
    want, got = _cache(device), _cache(device)
    want.append(0, key.to(device), value.to(device))
    expected = want.attend(0, q.to(device))
    mask = torch.rand((1, 1, 90, 3), generator=g).to(device).transpose(2, 3) < 0.5
    masked = want.attend(0, q.to(device), mask)
    k2, v2, q2 = swapped(key), swapped(value), swapped(q)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)
    ops.kv_append(got.blocks, 0, k2, v2, 0, stream=stream)
    outs = [ops.block_attention(got.blocks, 0, q2, 90, m, 0.125, stream=stream)
            for m in (None, mask)]
    none = ops.block_attention(got.blocks, 0, q2, 0, None, 0.125, stream=stream)
    with torch.cuda.stream(stream):
        copies = [t.clone() for t in (*outs, none)]
    stream.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(copies[0], expected) and torch.equal(copies[1], masked)
    assert not copies[2].any()


def test_token_numbers_past_32_bits_are_refused(device):
    cache = _cache(device)
    cache.append(0, *(torch.zeros((1, 2, 70, 64), dtype=torch.bfloat16, device=device),) * 2)
    q = torch.zeros((1, 2, 1, 64), dtype=torch.bfloat16, device=device)
    for keys in (-1, 2 ** 31, 2 ** 32 + 70):
        with pytest.raises(ValueError, match="keys"):
            ops.block_attention(cache.blocks, 0, q, keys, None, 1.0)
    for count in (-1, 9, 2 ** 32 + 1):
        with pytest.raises(ValueError, match="folded"):
            ops.kv_fold(cache.blocks, count)
    assert cache.folded_tokens == 0


def test_two_streams_at_once(device):
    """Calls that split their keys, each with scratch memory of its own."""
    g = torch.Generator().manual_seed(17)
    cache, _, _ = _filled(device, g, 1, 4, 128, 9000, 3, "int8")
    assert ops._block_attention_workspace(1, 3, 9003, 16, 4, 128) > 0
    qs = [_rand(g, 1, 16, 3, 128).to(device) for _ in range(2)]
    want = [cache.attend(0, q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    outs = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                outs[i].append(cache.attend(0, qs[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(o, want[i]) for o in outs[i])


@pytest.mark.parametrize("held,D,rows", [("e4m3", 128, 1), ("int8", 64, 80)])
def test_offsets_past_32_bits(device, held, D, rows):
    """The last head of a cache whose codes take more than 4 GiB, with the last
    blocks of a million tokens: appended, folded, read back and attended to."""
    heads, blocks = 40 * 128 // D, 16384
    start, new = (blocks - 3) * BLOCK, 150
    b = ops.KVBlocks(layers=1, batch=1, kv_heads=heads, head_dim=D, capacity_blocks=blocks,
                     ring_blocks=3, held=held, device=device)
    assert (heads - 1) * blocks * BLOCK * D > 2 ** 32
    b.keys.zero_()
    b.values.zero_()
    b.folded = blocks - 3
    g = torch.Generator().manual_seed(D)
    k, v, q = (_rand(g, 1, heads, n, D) for n in (new, new, rows))
    ops.kv_append(b, 0, k.to(device), v.to(device), start)
    ops.kv_fold(b, 2)
    got_k, got_v = ops.kv_read(b, 0, start, start + new)
    kk, vv = held_rows(k, 2, held), held_rows(v, 2, held)
    assert _same(got_k, kk) and _same(got_v, vv)
    # The tokens before are there and admit nobody.
    keys = start + new
    mask = torch.zeros((1, 1, rows, keys), dtype=torch.bool)
    mask[..., start:] = torch.rand((rows, new), generator=g) < 0.7
    mask[..., -1] = True
    out = ops.block_attention(b, 0, q.to(device), keys, mask.to(device), D ** -0.5)
    last = heads - 1
    want, bound = attention(q[:, last:], kk[:, last:], vv[:, last:], mask[..., start:], D ** -0.5)
    assert ((out[:, :, last:].cpu().double() - want).abs() <= bound).all()


def test_repeated_calls_give_the_same_bits(device):
    g = torch.Generator().manual_seed(14)
    for new, mask in ((1, None), (61, "tree"), (300, None)):
        cache, k, v = _filled(device, g, 1, 4, 128, 900, new, "e4m3")
        m = _mask(mask, g, 1, 900, new)
        m = None if m is None else m.to(device)
        q = _rand(g, 1, 32, new, 128).to(device)
        first = cache.attend(0, q, m)
        assert all(torch.equal(cache.attend(0, q, m), first) for _ in range(3))


def test_layers_are_apart(device):
    g = torch.Generator().manual_seed(15)
    layers, H, D, S = 3, 2, 64, 140
    cache = _cache(device, H=H, D=D, capacity=S, layers=layers, held="int8")
    rows = [(_rand(g, 1, H, S, D), _rand(g, 1, H, S, D)) for _ in range(layers)]
    for l, (k, v) in enumerate(rows):
        cache.append(l, k.to(device), v.to(device))
    cache.commit()
    for l, (k, v) in enumerate(rows):
        _check_attention(cache, _rand(g, 1, 4, 2, D), k, v, None, 0.125, "int8", layer=l)


def test_refusals(device):
    cache = _cache(device, H=2, D=64, capacity=200, tail=70)
    row = lambda n, h=2, d=64, t=torch.bfloat16: torch.zeros((1, h, n, d), dtype=t, device=device)  # noqa: E731
    with pytest.raises(ValueError, match="capacity|holds"):
        cache.append(0, row(201), row(201))
    with pytest.raises(ValueError, match="tail"):
        cache.append(0, row(200), row(200))
    with pytest.raises(ValueError, match="heads"):
        cache.append(0, row(4, h=3), row(4, h=3))
    with pytest.raises(ValueError, match="differ"):
        cache.append(0, row(4), row(5))
    with pytest.raises(ValueError, match="dtype"):
        cache.append(0, row(4, t=torch.float16), row(4))
    with pytest.raises(ValueError):
        cache.append(0, row(4, d=128), row(4, d=128))
    with pytest.raises(ValueError, match="device"):
        cache.append(0, row(4).cpu(), row(4).cpu())
    assert cache.get_seq_length() == 0
    cache.append(0, row(130), row(130))
    cache.commit()
    assert cache.folded_tokens == 128
    for length in (127, 0, -3):
        with pytest.raises(ValueError, match="folded"):
            cache.crop(length)
    cache.crop(129)
    with pytest.raises(ValueError, match="folded"):
        cache.compact(100, (3, 4))
    with pytest.raises(ValueError, match="ascend"):
        cache.compact(128, (0, 0))
    with pytest.raises(ValueError, match="ascend"):
        cache.compact(128, (1,))
    with pytest.raises(ValueError, match="length"):
        cache.compact(140, ())
    q = torch.zeros((1, 3, 2, 64), dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError, match="multiple"):
        cache.attend(0, q)
    q = torch.zeros((1, 4, 2, 64), dtype=torch.bfloat16, device=device)
    with pytest.raises(TypeError, match="bool"):
        cache.attend(0, q, torch.ones((1, 1, 2, 9), device=device))
    for shape in ((1, 1, 3, 9), (1, 2, 2, 9), (2, 1, 2, 9), (1, 1, 2, 130)):
        with pytest.raises(ValueError, match="mask"):
            cache.attend(0, q, torch.ones(shape, dtype=torch.bool, device=device))
    with pytest.raises(IndexError):
        ops.block_attention(cache.blocks, 1, q, 10, None, 1.0)
    with pytest.raises(RuntimeError, match="invalid argument"):
        ops.block_attention(cache.blocks, 0, q, 100000, None, 1.0)
    with pytest.raises(ValueError):
        cache.read(0, 5, 500)
    for bad in (dict(head_dim=80), dict(held="fp4"), dict(kv_heads=0), dict(device="cpu")):
        with pytest.raises(ValueError):
            BlockKVCache(**{**dict(layers=1, kv_heads=2, head_dim=64, capacity=64, device=device),
                            **bad})
