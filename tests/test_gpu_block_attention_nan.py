"""What is not finite in queries and keys of the block attention (K10), in every
form it takes.  The softmax is NaN where one of a row's admitted scores is NaN, or
where all of them are -inf; a row is zeros only where it admits no key, and a row
that does not admit a bad key keeps its bits."""
import math

import pytest
import torch

from _block_forms import ONE_OF_EACH
from specfit_amd.runtime import BlockKVCache

pytestmark = pytest.mark.gpu

# batch, query heads, KV heads, D, queries, keys
CASES = [(1, 8, 2, 128, 1, 27), (1, 8, 2, 128, 1, 65), (1, 8, 2, 64, 1, 129), (1, 4, 2, 64, 30, 30),
         (2, 8, 2, 128, 61, 500), (1, 32, 1, 128, 64, 2000), (8, 64, 4, 128, 32, 32),
         (3, 256, 1, 64, 32, 32), (4, 32, 4, 128, 256, 256), (1, 32, 4, 128, 300, 2300)]
CASES += [c for c in ONE_OF_EACH.values() if c not in CASES]
IDS = ["x".join(map(str, c)) for c in CASES]


def _inputs(case, seed=0):
    B, Hq, H, D, Q, S = case
    g = torch.Generator().manual_seed(seed)
    return [torch.randn((B, h, n, D), generator=g).to(torch.bfloat16)
            for h, n in ((Hq, Q), (H, S), (H, S))]


def _attend(device, case, q, k, v, mask=None, held="e4m3"):
    """The last token is in bf16, and so are those of its block."""
    B, _, H, D, _, S = case
    cache = BlockKVCache(1, H, D, S, batch=B, held=held, tail_tokens=S, device=device)
    folded = (S - 1) // 64 * 64
    if folded:
        cache.append(0, k[:, :, :folded].to(device), v[:, :, :folded].to(device))
        cache.commit()
    cache.append(0, k[:, :, folded:].to(device), v[:, :, folded:].to(device))
    return cache.attend(0, q.to(device), None if mask is None else mask.to(device)).cpu()


def _check(out, clean, bad):
    """NaN in the rows `bad` (bool [B, Q, Hq]), the bits of `clean` in the others."""
    assert bool(out[bad].isnan().all())
    assert torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("masked", (False, True))
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_nan_queries(device, case, masked):
    B, Hq, _, _, Q, S = case
    q, k, v = _inputs(case)
    g = torch.Generator().manual_seed(1)
    mask = None
    if masked:
        mask = torch.rand((B, 1, Q, S), generator=g) < 1.5 / S  # a key or two, or none
        admits = mask.any(-1)[:, 0, :, None].expand(B, Q, Hq)
    else:
        admits = torch.ones((B, Q, Hq), dtype=torch.bool)
    clean = _attend(device, case, q, k, v, mask)
    assert bool(clean.isfinite().all()) and not clean[~admits].any()
    bad = torch.rand((B, Q, Hq), generator=g) < 0.2
    bad[:, 0, 0] = True
    q[bad.transpose(1, 2)] = math.nan
    _check(_attend(device, case, q, k, v, mask), clean, bad & admits)


@pytest.mark.parametrize("held", ("e4m3", "int8"))
@pytest.mark.parametrize("where", ("first", "last"))
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_a_nan_key(device, case, where, held):
    """In every mask's reach (causal), and as the only key of some rows."""
    B, Hq, H, _, Q, S = case
    q, k, v = _inputs(case)
    place = 0 if where == "first" else S - 1
    k[-1, -1, place, 5] = 0.0  # the block's scale is that of its finite values
    damaged = k.clone()
    damaged[-1, -1, place, 5] = math.nan
    heads = torch.zeros((B, Q, Hq), dtype=torch.bool)
    heads[-1, :, Hq - Hq // H:] = True
    sees = torch.arange(S)[None] <= S - Q + torch.arange(Q)[:, None]
    bad = heads & sees[:, place, None]
    _check(_attend(device, case, q, damaged, v, None, held), _attend(device, case, q, k, v, None, held),
           bad)
    mask = torch.zeros((1, 1, Q, S), dtype=torch.bool)
    mask[..., ::3, :] = torch.rand((len(range(0, Q, 3)), S),
                                   generator=torch.Generator().manual_seed(2)) < 0.3
    mask[..., ::3, place] = False
    mask[..., 1::3, place] = True  # only the bad key; the rows in between admit nothing
    if Q == 1:
        mask[..., place] = True
    bad = heads & mask[0, 0, :, place, None]
    clean = _attend(device, case, q, k, v, mask, held)
    assert not clean[:, 2::3].any()
    _check(_attend(device, case, q, damaged, v, mask, held), clean, bad)


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_scores_of_minus_infinity(device, case):
    """A key whose score is -inf counts for nothing beside others; a row that
    admits no others has no softmax."""
    B, Hq, H, _, Q, S = case
    q, k, v = _inputs(case)
    q[..., 0] = q[..., 0].abs() + 1
    damaged = k.clone()
    damaged[:, :, S - 1, 0] = -math.inf
    mask = torch.rand((1, 1, Q, S), generator=torch.Generator().manual_seed(3)) < 0.5
    mask[..., 0] = True
    mask[..., S - 1] = False
    clean = _attend(device, case, q, k, v, mask)
    mask[..., S - 1] = True
    mask[..., 1::2, :S - 1] = False
    if Q > 4:
        mask[..., 3, :] = False
    alone = (mask.sum(-1) == 1)[0, 0, :, None].expand(B, Q, Hq)
    out = _attend(device, case, q, damaged, v, mask)
    clean[:, 1::2] = 0.0
    if Q > 4:
        clean[:, 3] = 0.0
    _check(out, clean, alone)
    if Q == 1:
        mask[..., :S - 1] = False
        assert bool(_attend(device, case, q, damaged, v, mask).isnan().all())
