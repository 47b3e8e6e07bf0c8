"""Plain 64-bit forms of the block cache and its attention, on the CPU."""
import math

import torch

BLOCK = 64
EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half steps


def fold(x: torch.Tensor, held: str):
    """x [..., 64, D] (one block each, any float type) -> (x^ float64, scale
    float64 [...]): the least 2^e, e >= -60, with max |finite x| <= q 2^e; codes
    to the nearest, ties to even; what is not finite as NaN."""
    x = x.double()
    finite = torch.isfinite(x)
    top = torch.where(finite, x, torch.zeros_like(x)).abs().amax(dim=(-2, -1))
    q = 127.0 if held == "int8" else 448.0
    e = torch.full(top.shape, -60.0, dtype=torch.float64)
    while bool((top > q * torch.exp2(e)).any()):
        e = torch.where(top > q * torch.exp2(e), e + 1, e)
    scale = torch.exp2(e)
    y = torch.where(finite, x, torch.zeros_like(x)) / scale[..., None, None]
    if held == "int8":
        y = torch.round(y)
    else:  # e4m3: 3 bits behind the leading one, subnormal below 2^-6
        _, p = torch.frexp(y)
        step = torch.exp2((p - 1).clamp_min(-6).double() - 3)
        y = torch.round(y / step) * step
    y = y * scale[..., None, None]
    return torch.where(finite, y, torch.full_like(y, math.nan)), scale


def held_rows(x: torch.Tensor, folded: int, held: str):
    """x [B, H, S, D] as the cache gives it back with ``folded`` blocks
    folded, float64."""
    x = x.cpu().double()
    n = folded * BLOCK
    if n == 0:
        return x
    blocks, _ = fold(x[:, :, :n].unflatten(2, (folded, BLOCK)), held)
    return torch.cat([blocks.flatten(2, 3), x[:, :, n:]], dim=2)


def admit_matrix(mask, B, Q, S):
    """bool [B, Q, S]."""
    if mask is None:
        return (torch.arange(S)[None] <= S - Q + torch.arange(Q)[:, None]).expand(B, Q, S)
    mask = mask.cpu()
    admit = torch.ones((B, Q, S), dtype=torch.bool)
    admit[:, :, S - mask.shape[-1]:] = mask[:, 0].expand(B, -1, -1)
    return admit


def attention(q, k, v, mask, scale):
    """q [B, Hq, Q, D], k and v [B, H, S, D] float64 -> (out [B, Q, Hq, D], bound
    of a kernel with fp32 scores, weights rounded to bf16 and a bf16 result).

    The bound: each weight is off by half a bf16 step of itself, by its score's
    error and by that of the exponential.  A score is a sum of D products whose
    roundings (2^-24 each, D + 2 of them with the factors) are relative to
    sum |q k|; the reference taken off in log2 units, at most 8 above the largest
    score, and the product with the factor add 2 steps of the largest score and of 8
    (2^-24 8 = 2^-21 each); the value scale's exponent, of at most 128, joins the
    reference in one more sum (2^-24 128 = 2^-17); an exponential is good to 2^-21;
    these together stay below 2^-16.
    The sum of the weights has the same but for the bf16 step.  The result is
    rounded once.  A key whose weight times the value scale 2^e falls below 2^-126
    (fp32's least normal number) may count for nothing: its part is below 2^-126
    |code| <= 2^-126 448 < 2^-117, S of them below S 2^-117, over a sum of weights of
    at least 2^-8."""
    q = q.cpu().double()
    B, Hq, Q, D = q.shape
    H, S = k.shape[1], k.shape[2]
    admit = admit_matrix(mask, B, Q, S)
    out = torch.zeros((B, Q, Hq, D), dtype=torch.float64)
    bound = torch.zeros_like(out)
    for b in range(B):
        for h in range(Hq):
            kk, vv = k[b, h // (Hq // H)], v[b, h // (Hq // H)]
            s = (q[b, h] @ kk.T) * scale
            mag = (q[b, h].abs() @ kk.abs().T) * abs(scale)
            s = torch.where(admit[b], s, torch.full_like(s, -math.inf))
            mag = torch.where(admit[b], mag, torch.zeros_like(mag))
            some = admit[b].any(1)
            top = torch.where(some[:, None], s.amax(1, keepdim=True), torch.zeros(Q, 1).double())
            p = torch.exp(s - top)
            p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
            out[b, :, h] = p @ vv
            size = p @ vv.abs()
            weight = 2.0 ** -24 * ((D + 2) * mag.amax(1) + 4 * mag.amax(1)) * 2 + 2.0 ** -16
            bound[b, :, h] = (EPS[torch.bfloat16] + weight)[:, None] * size \
                + EPS[torch.bfloat16] * (1 + EPS[torch.bfloat16]) * out[b, :, h].abs() + S * 2.0 ** -109
    return out, bound
