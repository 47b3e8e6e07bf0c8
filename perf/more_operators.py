"""Operators of layers held in microscaled 4 bits, their plain forms and the
calls whose speed matters.

    kind      operator                                           entry points
    quantize  activations to e4m3 and weights to e2m1 in blocks   ops.mx_quantize / mx_quantize_weight
              of 32 with a power-of-two scale, and their values
    norm      the residual's addition, RMSNorm, and its output    ops.add_rms_norm
              in e4m3 with scales besides
    linear    activations in e4m3 times weights in e2m1           ops.mx_linear
    experts   routed SwiGLU experts with weights in e2m1          runtime.Qwen3MXExperts

A block of 32 neighbours in a row shares the scale 2^e, e the smallest integer
from -127 up at which no value rounds past the type's largest (448, 6). Values
are rounded to the nearest, ties to even.

With ``own`` false, ``run`` computes each in elementary torch operations in
32 bits; with ``own`` true it makes the framework's calls.  ``exact`` computes
the definitions in 64 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
BLOCK = 32
EPS = 1e-6
VOCAB = 151936
TYPES = ("bfloat16", "float16", "float32")


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # The attention outputs of a 60-node draft tree and its seed, before
        # the output projection.
        dict(name="quantize_tree", kind="quantize", form="rows", rows=61, dim=4096, dtype="bfloat16"),
        # A long prompt's activations.
        dict(name="quantize_prompt", kind="quantize", form="rows", rows=8192, dim=4096,
             dtype="bfloat16"),
        # A model's output embedding when it is loaded.
        dict(name="quantize_head", kind="quantize", form="weight", rows=VOCAB, dim=2048,
             dtype="bfloat16"),
        # One decoded token between attention and experts.
        dict(name="norm_decode", kind="norm", rows=1, dim=2048, residual=True, dtype="bfloat16"),
        # A prompt's rows at a model's first layer: no residual yet, odd width.
        dict(name="norm_odd", kind="norm", rows=1333, dim=1001, residual=False, dtype="float32"),
        # A long prompt, in a wide model.
        dict(name="norm_prompt", kind="norm", rows=8192, dim=4096, residual=True, dtype="bfloat16"),
        # One decoded token's queries, keys and values.
        dict(name="linear_decode", kind="linear", rows=1, dim=2048, out=5120, x="tensor", bias=False,
             dtype="bfloat16"),
        # The logits of a draft tree's rows.
        dict(name="linear_tree_head", kind="linear", rows=61, dim=2048, out=VOCAB, x="rows",
             bias=False, dtype="bfloat16"),
        # Queries, keys and values of a prompt, in a wide model.
        dict(name="linear_prompt", kind="linear", rows=4096, dim=4096, out=9216, x="rows", bias=False,
             dtype="bfloat16"),
        # One decoded token's experts.
        dict(name="experts_decode", kind="experts", tokens=1, hidden=2048, inner=768, experts=128,
             top_k=8, zipf=0.0),
        # A draft tree's experts, some of them favourites.
        dict(name="experts_tree", kind="experts", tokens=61, hidden=2048, inner=768, experts=128,
             top_k=8, zipf=1.1),
        # A prompt chunk's experts.
        dict(name="experts_prompt", kind="experts", tokens=2048, hidden=2048, inner=768, experts=128,
             top_k=8, zipf=0.0),
    ]


def _log(rng, low, high):
    high = max(low, high)
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng: random.Random):
    kind = rng.choice(["quantize", "norm", "linear", "linear", "experts", "experts"])
    dtype = rng.choice(TYPES)
    if kind == "quantize":
        dim = rng.choice([2048, 4096, _log(rng, 8, 12000)])
        return dict(kind=kind, form=rng.choice(["rows", "weight"]),
                    rows=_log(rng, 1, min(100000, 100_000_000 // dim)), dim=dim, dtype=dtype)
    if kind == "norm":
        dim = rng.choice([128, 2048, 4096, _log(rng, 16, 12000)])
        return dict(kind=kind, rows=_log(rng, 1, min(20000, 16_000_000 // dim)), dim=dim,
                    residual=rng.random() < 0.6, dtype=dtype)
    if kind == "linear":
        dim = rng.choice([768, 2048, 4096, _log(rng, 40, 8000)])
        rows = rng.choice([1, _log(rng, 2, 200), _log(rng, 64, 4096)])
        out = _log(rng, 24, 50000)
        while rows * dim * out > 140e9:
            out = out // 2 + 1
        return dict(kind=kind, rows=rows, dim=dim, out=out, x=rng.choice(["tensor", "rows"]),
                    bias=rng.random() < 0.3, dtype=rng.choice(["bfloat16", "bfloat16", "float16"]))
    hidden, inner, most, top_k = rng.choice([(2048, 768, 128, 8), (2048, 768, 128, 8),
                                             (4096, 1536, 32, 8), (64, 32, 256, 3),
                                             (1000, 424, 100, 2)])
    experts = _log(rng, top_k, most)
    most = min(2048, int(150e9 / (6 * hidden * inner * top_k)))
    return dict(kind=kind, tokens=rng.choice([_log(rng, 1, 100), _log(rng, 1, most)]), hidden=hidden,
                inner=inner, experts=experts, top_k=top_k, zipf=rng.choice([0.0, 1.1]))


# ----------------------------------------------------------------- inputs --
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _activations(g, rows, dim):
    """Rows of different sizes with a few loud channels, as a residual stream
    has."""
    loud = torch.ones(dim, device=DEV)
    loud[dim // 3], loud[dim // 2] = 30.0, 12.0
    return _normal(g, rows, dim) * loud * torch.exp(0.5 * _normal(g, rows, 1))


def _inputs(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    if kind == "quantize":
        if case["form"] == "rows":
            x = _activations(g, case["rows"], case["dim"])
        else:
            x = 0.02 * _normal(g, case["rows"], case["dim"])
        return dict(x=x.to(getattr(torch, case["dtype"])))
    if kind == "norm":
        dtype, rows, dim = getattr(torch, case["dtype"]), case["rows"], case["dim"]
        x = _activations(g, rows, dim).to(dtype)
        return dict(x=x, residual=_activations(g, rows, dim).to(dtype) if case["residual"] else None,
                    weight=(1.0 + 0.2 * _normal(g, dim)).to(dtype))
    if kind == "linear":
        dtype = getattr(torch, case["dtype"])
        x = _activations(g, case["rows"], case["dim"]).to(dtype)
        w = (0.02 * _normal(g, case["out"], case["dim"])).to(dtype)
        return dict(x=x, w=w, bias=_normal(g, case["out"]).to(dtype) if case["bias"] else None)
    t, h, i, e, k = (case[n] for n in ("tokens", "hidden", "inner", "experts", "top_k"))
    # Tokens after a norm, experts as [gate | up | down].
    hidden = _normal(g, t, h).to(torch.bfloat16)
    packed = torch.empty((e, 3 * h * i), dtype=torch.bfloat16, device=DEV).normal_(0, 0.02, generator=g)
    logits = -case["zipf"] * torch.log(torch.arange(1, e + 1, device=DEV).float())
    logits = logits[torch.randperm(e, generator=g, device=DEV)]
    u = torch.rand((t, e), generator=g, device=DEV).clamp_(1e-9, 1 - 1e-7)
    scores, index = torch.topk(logits - torch.log(-torch.log(u)), k, dim=1)
    weights = torch.softmax(scores, dim=1).to(torch.bfloat16)
    return dict(hidden=hidden, packed=packed, index=index, weights=weights)


# -------------------------------------------------------------- plain forms --
def _plain_blocks(x, held):
    """x [..., K] -> values of the codes [..., n, 32] and scale exponents [..., n]."""
    k = x.shape[-1]
    y = torch.nn.functional.pad(x.float(), (0, -k % BLOCK)).unflatten(-1, (-1, BLOCK))
    m, e = torch.frexp(y.abs().amax(-1))
    if held == "e4m3":   # up to 464 rounds to 448
        e = torch.where(m <= 464 / 512, e - 9, e - 8)
    else:                # below 7 rounds to 6
        e = torch.where(m < 7 / 8, e - 3, e - 2)
    e = torch.where(m == 0, -127, e).clamp_min(-127)
    y = torch.ldexp(y, -e[..., None])
    if held == "e4m3":
        return y.to(torch.float8_e4m3fn).float(), e
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    return torch.round(y / step) * step, e


def _plain_values(codes, e, k):
    return torch.ldexp(codes, e[..., None]).flatten(-2)[..., :k]


FOUR_BITS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _plain_pack(w):
    """A weight as a program keeps it: two codes to a byte, and scale bytes."""
    values, e = _plain_blocks(w, "e2m1")
    sizes = torch.tensor(FOUR_BITS, device=DEV)
    code = torch.bucketize(values.abs(), sizes).to(torch.uint8) | ((values < 0).to(torch.uint8) << 3)
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _plain_unpack(codes, scales, k):
    table = torch.tensor(FOUR_BITS + tuple(-x for x in FOUR_BITS), device=DEV)
    pairs = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).unflatten(-1, (-1, BLOCK))
    return _plain_values(table[pairs.int()], scales.int() - 127, k)


def _plain_quantize(s):
    held = "e4m3" if s["form"] == "rows" else "e2m1"
    return _plain_values(*_plain_blocks(s["x"], held), s["x"].shape[-1]).to(torch.bfloat16)


def _plain_norm(s):
    x, dtype = s["x"], s["x"].dtype
    if s["residual"] is not None:
        x = (x.float() + s["residual"].float()).to(dtype)
    # The mean of squares in 64 bits: 8-bit codes lie on borders.
    r = torch.rsqrt(x.double().square().mean(-1, keepdim=True) + EPS).float()
    y = x.float() * r * s["weight"].float()
    q = _plain_values(*_plain_blocks(y, "e4m3"), y.shape[-1]).to(torch.bfloat16)
    return {"sum": x, "normed": y.to(dtype), "quantized": q}


def _plain_linear(s):
    if "x8" in s:
        x = _plain_values(s["x8"].float(), s["x_scale"], s["dim"])
    else:
        x = _plain_values(*_plain_blocks(s["x"], "e4m3"), s["dim"])
    y = x @ _plain_unpack(*s["w4"], s["dim"]).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["dtype"])


def _plain_experts(s):
    hidden, index, weights = s["hidden"], s["index"], s["weights"].float()
    (t, h), k, i = hidden.shape, index.shape[1], s["inner"]
    x = _plain_values(*_plain_blocks(hidden, "e4m3"), h)
    # The routes in order of expert, each expert's rows padded to the most that one has.
    expert, order = torch.sort(index.flatten(), stable=True)
    active, at, count = torch.unique_consecutive(expert, return_inverse=True, return_counts=True)
    place = torch.arange(t * k, device=DEV) - (torch.cumsum(count, 0) - count)[at]
    rows = torch.zeros((active.numel(), int(count.max()), h), device=DEV)
    rows[at, place] = x[order // k]
    gate, up, down = (_plain_unpack(codes[active], scales[active], width).transpose(1, 2).contiguous()
                      for (codes, scales), width in zip(s["w4"], (h, h, i)))
    g = torch.bmm(rows, gate)
    act = g / (1 + torch.exp(-g)) * torch.bmm(rows, up)
    act = _plain_values(*_plain_blocks(act, "e4m3"), i)
    y = torch.bmm(act, down)[at, place] * weights.flatten()[order, None]
    out = torch.zeros((t * k, h), device=DEV)
    out[order] = y
    return out.view(t, k, h).sum(1).to(torch.bfloat16)


# --------------------------------------------------------- prepare and run --
def prepare(case, seed):
    s = _inputs(case, seed)
    kind = s["kind"] = case["kind"]
    if kind == "quantize":
        s["form"] = case["form"]
    elif kind == "linear":
        s["dim"], s["dtype"] = case["dim"], s["x"].dtype
        w = s.pop("w")
        if own:
            from specfit_amd import ops
            s["weight"] = ops.mx_quantize_weight(w)
            if case["x"] == "rows":  # as a norm leaves them
                s["x"] = ops.mx_quantize(s["x"])
        else:
            s["w4"] = _plain_pack(w)
            if case["x"] == "rows":
                codes, s["x_scale"] = _plain_blocks(s.pop("x"), "e4m3")
                s["x8"] = codes.to(torch.float8_e4m3fn)
    elif kind == "experts":
        s["inner"] = i = case["inner"]
        e, h, packed = case["experts"], case["hidden"], s.pop("packed")
        if own:
            from specfit_amd.runtime import Qwen3MXExperts
            s["experts"] = Qwen3MXExperts.from_packed(packed, hidden_size=h, intermediate_size=i)
        else:
            gate, up, down = packed.split(h * i, dim=1)
            s["w4"] = [_plain_pack(gate.view(e, i, h)), _plain_pack(up.view(e, i, h)),
                       _plain_pack(down.reshape(e, h, i))]
    return s


def run(state):
    s, kind = state, state["kind"]
    if not own:
        return {"quantize": _plain_quantize, "norm": _plain_norm, "linear": _plain_linear,
                "experts": _plain_experts}[kind](s)
    from specfit_amd import ops
    if kind == "quantize":
        if s["form"] == "rows":
            return ops.mx_quantize(s["x"]).values()
        return ops.mx_quantize_weight(s["x"]).values()
    if kind == "norm":
        total, normed, rows = ops.add_rms_norm(s["x"], s["residual"], s["weight"], EPS,
                                               quantized=True)
        return {"sum": total, "normed": normed, "quantized": rows.values()}
    if kind == "linear":
        return ops.mx_linear(s["x"], s["weight"], s["bias"])
    return s["experts"](s["hidden"], s["index"], s["weights"])


# ------------------------------------------------------------------- work --
def _held_bytes(rows, dim, bits):
    return rows * (dim * bits // 8 + (dim + BLOCK - 1) // BLOCK)


def work(case):
    kind = case["kind"]
    if kind == "quantize":
        n = case["rows"] * case["dim"]
        size = 4 if case["dtype"] == "float32" else 2
        held = _held_bytes(case["rows"], case["dim"], 8 if case["form"] == "rows" else 4)
        # Read, held, read back, and the values written.
        return {"bytes": n * size + 2 * held + 2 * n, "flops": 4 * n}
    if kind == "norm":
        n = case["rows"] * case["dim"]
        size = 4 if case["dtype"] == "float32" else 2
        # Without a residual the sum is the input itself.
        moved = n * size * (4 if case["residual"] else 2) + size * case["dim"]
        return {"bytes": moved + 2 * _held_bytes(case["rows"], case["dim"], 8) + 2 * n,
                "flops": 8 * n}
    if kind == "linear":
        m, k, n = case["rows"], case["dim"], case["out"]
        read = _held_bytes(m, k, 8) if case["x"] == "rows" else 2 * m * k
        return {"bytes": read + _held_bytes(n, k, 4) + 2 * m * n + (2 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    t, h, i, e, k = (case[n] for n in ("tokens", "hidden", "inner", "experts", "top_k"))
    share = [(j + 1) ** -case["zipf"] for j in range(e)]
    hit = sum(1 - (1 - min(1.0, k * p / sum(share))) ** t for p in share)  # experts with a token
    expert = 2 * _held_bytes(i, h, 4) + _held_bytes(h, i, 4)
    return {"bytes": int(hit * expert) + 4 * t * h + 10 * t * k, "flops": 6 * t * k * h * i}


# ------------------------------------------------------------------ exact --
def _exact_values(x, held):
    """x [rows, K] in 64 bits -> the values that blocks of 32 hold of it."""
    rows, k = x.shape
    lowest, bits, past = (-6.0, 3.0, 464.0) if held == "e4m3" else (0.0, 1.0, 7.0)
    out = torch.empty_like(x)
    for begin in range(0, rows, 16384):
        part = x[begin:begin + 16384]
        blocks = torch.zeros((part.shape[0], (k + BLOCK - 1) // BLOCK * BLOCK), dtype=torch.float64,
                             device=x.device)
        blocks[:, :k] = part
        blocks = blocks.view(part.shape[0], -1, BLOCK)
        top = blocks.abs().amax(2, keepdim=True)
        # A guess that is too small by one or two, then up while the largest is past the type's.
        scale = torch.exp2(torch.floor(torch.log2(top.clamp_min(1e-300) / past)) - 1)
        for _ in range(3):
            over = top > past * scale if held == "e4m3" else top >= past * scale
            scale = torch.where(over, 2 * scale, scale)
        scale = scale.clamp_min(2.0 ** -127)
        y = blocks / scale
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** lowest))) - bits)
        y = torch.round(y / step) * step * scale
        out[begin:begin + 16384] = y.view(part.shape[0], -1)[:, :k]
    return out


def exact(case, seed):
    s, kind = _inputs(case, seed), case["kind"]
    if kind == "quantize":
        return _exact_values(s["x"].double(), "e4m3" if case["form"] == "rows" else "e2m1")
    if kind == "norm":
        x = s["x"].double()
        if s["residual"] is not None:
            x = (x + s["residual"].double()).to(s["x"].dtype).double()  # held in the stream's type
        y = x / torch.sqrt((x * x).sum(1, keepdim=True) / x.shape[1] + EPS) * s["weight"].double()
        return {"sum": x, "normed": y, "quantized": _exact_values(y, "e4m3")}
    if kind == "linear":
        x = _exact_values(s["x"].double(), "e4m3")
        parts = [x @ _exact_values(w.double(), "e2m1").t() for w in s["w"].split(16384)]
        y = torch.cat(parts, dim=1)
        return y if s["bias"] is None else y + s["bias"].double()
    h, i, k = case["hidden"], case["inner"], case["top_k"]
    x = _exact_values(s["hidden"].double(), "e4m3")
    out = torch.zeros_like(x)
    for e in range(case["experts"]):
        token, slot = torch.nonzero(s["index"] == e, as_tuple=True)
        if not token.numel():
            continue
        gate, up, down = s["packed"][e].double().split(h * i)
        g = x[token] @ _exact_values(gate.view(i, h), "e2m1").t()
        act = g * torch.sigmoid(g) * (x[token] @ _exact_values(up.view(i, h), "e2m1").t())
        y = _exact_values(act, "e4m3") @ _exact_values(down.view(h, i), "e2m1").t()
        out.index_add_(0, token, y * s["weights"][token, slot].double()[:, None])
    return out
