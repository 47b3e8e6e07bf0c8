"""Operators of the verification step around its sequence, their plain forms
and the calls whose speed matters.

    kind      operator                                          entry points
    attend    new keys and values appended to a cache whose      runtime.BlockKVCache.append / attend
              complete blocks are held in 8 bits, and attention
              over it
    fold      a prompt or an accepted draft path into the 8-bit  BlockKVCache.append / compact / commit / read
              blocks, and the cache's content read back
    rotary    rotary positions of queries and keys               ops.rotary_embed
    rules     repetition penalties, biases and grammar masks     runtime.LogitRules.adjust / greedy
              on the logits of a draft tree's rows

With ``own`` false, ``run`` computes each in elementary torch operations in
32 bits; with ``own`` true it makes the framework's calls.  ``exact`` computes
the definitions in 64 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
BLOCK = 64          # tokens of a cache block: one scale per block, head and K or V
MIN_EXPONENT = -60  # of a block's power-of-two scale
VOCAB = 151936


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # One decoded token over a short conversation: all latency.
        dict(name="attend_decode_short", kind="attend", batch=1, q_heads=32, kv_heads=4, dim=128,
             prefix=200, new=1, mask="causal", held="e4m3"),
        # One decoded token over a long document.
        dict(name="attend_decode_long", kind="attend", batch=1, q_heads=32, kv_heads=4, dim=128,
             prefix=131071, new=1, mask="causal", held="int8"),
        # The verification of a 60-node draft tree and its seed.
        dict(name="attend_tree", kind="attend", batch=1, q_heads=32, kv_heads=4, dim=128,
             prefix=1024, new=61, mask="tree", held="e4m3"),
        # A 127-node draft tree on 64 query heads, deep into a long context.
        dict(name="attend_tree_far", kind="attend", batch=1, q_heads=64, kv_heads=4, dim=128,
             prefix=32777, new=128, mask="tree", held="int8"),
        # A chunk of a long prompt after what came before it.
        dict(name="attend_prompt", kind="attend", batch=1, q_heads=32, kv_heads=4, dim=128,
             prefix=16000, new=2048, mask="causal", held="e4m3"),
        # Sixteen left-padded sequences decoded together, small heads; the
        # last one is padding throughout.
        dict(name="attend_batch", kind="attend", batch=16, q_heads=16, kv_heads=4, dim=64,
             prefix=5000, new=3, mask="padded", held="int8"),
        # A prompt into the cache.
        dict(name="fold_prompt", kind="fold", batch=1, kv_heads=4, dim=128, tokens=8192, tree=0,
             kept=0, held="e4m3"),
        # Six of a tree's 61 nodes accepted, which completes a block.
        dict(name="fold_tree", kind="fold", batch=1, kv_heads=4, dim=128, tokens=123, tree=61,
             kept=6, held="int8"),
        # One decoded token's query and key.
        dict(name="rotary_decode", kind="rotary", batch=1, tokens=1, q_heads=32, kv_heads=4,
             dim=128, rotary=128, interleaved=False, scaling="none", dtype="bfloat16",
             start=32767),
        # A prompt chunk far into a stretched context, half of each head
        # rotated in pairs of neighbours.
        dict(name="rotary_prompt", kind="rotary", batch=2, tokens=4001, q_heads=32, kv_heads=4,
             dim=128, rotary=64, interleaved=True, scaling="yarn", dtype="float32", start=100000),
        # The greedy tokens of a 61-row draft tree under a grammar.
        dict(name="rules_greedy_tree", kind="rules", rows=61, vocab=VOCAB, depth=9, seen=4000,
             bias=False, grammar=True, repetition=1.1, presence=0.25, frequency=0.125,
             output="tokens", dtype="bfloat16"),
        # One row's adjusted logits for a sampler, with a bias.
        dict(name="rules_adjust_row", kind="rules", rows=1, vocab=32001, depth=1, seen=1000,
             bias=True, grammar=False, repetition=1.3, presence=0.0, frequency=0.5,
             output="logits", dtype="float32"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng: random.Random):
    kind = rng.choice(["attend", "attend", "attend", "fold", "rotary", "rules"])
    held = rng.choice(["e4m3", "int8"])
    if kind == "attend":
        q_heads, kv_heads, dim = rng.choice([(32, 4, 128), (64, 4, 128), (16, 4, 64), (8, 8, 64),
                                             (12, 4, 128), (14, 2, 64), (40, 8, 128)])
        mask = rng.choice(["causal", "causal", "tree", "padded"])
        if mask == "causal" and rng.random() < 0.5:      # one decoded token
            new, prefix, batch = 1, _log(rng, 16, 100000), rng.choice([1, 1, 2, 5])
        elif mask == "causal":                           # a prompt chunk
            new, prefix, batch = _log(rng, 65, 2000), rng.choice([0, _log(rng, 16, 12000)]), 1
        elif mask == "tree":
            new, prefix, batch = _log(rng, 2, 160), _log(rng, 16, 30000), 1
        else:
            new, prefix, batch = _log(rng, 1, 40), _log(rng, 16, 4000), rng.randint(2, 16)
        return dict(kind=kind, batch=batch, q_heads=q_heads, kv_heads=kv_heads, dim=dim,
                    prefix=prefix, new=new, mask=mask, held=held)
    if kind == "fold":
        tokens = _log(rng, 1, 8000)
        tree = rng.choice([0, min(tokens, _log(rng, 1, 160))])
        return dict(kind=kind, batch=rng.choice([1, 1, 2, 3]), kv_heads=rng.choice([1, 2, 4, 8]),
                    dim=rng.choice([64, 128]), tokens=tokens, tree=tree,
                    kept=rng.randint(1, min(tree, 20)) if tree else 0, held=held)
    if kind == "rotary":
        dim = rng.choice([64, 80, 128, 256])
        return dict(kind=kind, batch=rng.choice([1, 1, 2, 4]), tokens=_log(rng, 1, 3000),
                    q_heads=rng.choice([8, 14, 32]), kv_heads=rng.choice([1, 2, 4, 8]), dim=dim,
                    rotary=rng.choice([dim, dim // 2, 16]), interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "llama3", "yarn"]),
                    dtype=rng.choice(["bfloat16", "float16", "float32"]),
                    start=_log(rng, 1, 1000000))
    rows = _log(rng, 1, 160)
    return dict(kind=kind, rows=rows, vocab=rng.choice([VOCAB, 32001, 50257, _log(rng, 100, 150000)]),
                depth=rng.randint(1, 12), seen=_log(rng, 1, 20000), bias=rng.random() < 0.5,
                grammar=rng.random() < 0.5, repetition=rng.choice([1.0, 1.05, 1.1, 1.3]),
                presence=rng.choice([0.0, 0.25, 0.7]), frequency=rng.choice([0.0, 0.1, 0.5]),
                output=rng.choice(["tokens", "logits"]),
                dtype=rng.choice(["bfloat16", "float16", "float32"]))


# ----------------------------------------------------------------- inputs --
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _key_value(g, batch, heads, tokens, dim):
    """Keys with a few loud channels (as trained keys have) and values."""
    loud = torch.ones(dim, device=DEV)
    loud[3], loud[dim // 2 + 5] = 6.0, 4.0
    k = (_normal(g, batch, heads, tokens, dim) * loud).to(torch.bfloat16)
    # Tokens differ in size, so blocks differ in scale.
    size = torch.exp(0.5 * _normal(g, batch, heads, (tokens + 15) // 16, 1))
    size = size.repeat_interleave(16, dim=2)[:, :, :tokens]
    v = (_normal(g, batch, heads, tokens, dim) * size).to(torch.bfloat16)
    return k, v


def _attend_inputs(case, seed):
    g = _generator(seed)
    b, new, prefix = case["batch"], case["new"], case["prefix"]
    k, v = _key_value(g, b, case["kv_heads"], prefix + new, case["dim"])
    q = _normal(g, b, case["q_heads"], new, case["dim"]).to(torch.bfloat16)
    mask = None
    if case["mask"] == "tree":  # over the new keys: each node's ancestors and itself
        at = random.Random(seed)
        m = torch.eye(new, dtype=torch.bool)
        for i in range(1, new):
            m[i] |= m[at.randrange(max(0, i - 12), i)]
        mask = m.view(1, 1, new, new).to(DEV)
    elif case["mask"] == "padded":  # left padding; the last sequence is nothing but padding
        at = random.Random(seed)
        keys = prefix + new
        pad = torch.tensor([at.randrange(0, prefix) for _ in range(b - 1)] + [keys], device=DEV)
        s = torch.arange(keys, device=DEV)
        causal = s[None, :] <= prefix + torch.arange(new, device=DEV)[:, None]
        mask = (causal[None] & (s[None, None, :] >= pad[:, None, None])).view(b, 1, new, keys)
    return dict(k=k, v=v, q=q, mask=mask, scale=case["dim"] ** -0.5)


def _fold_inputs(case, seed):
    g = _generator(seed)
    k, v = _key_value(g, case["batch"], case["kv_heads"], case["tokens"], case["dim"])
    kept = tuple(sorted(random.Random(seed).sample(range(case["tree"]), case["kept"])))
    return dict(k=k, v=v, base=case["tokens"] - case["tree"], kept=kept)


SCALINGS = {
    "none": None,
    "linear": dict(rope_type="linear", factor=4.0),
    "llama3": dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                   original_max_position_embeddings=8192),
    "yarn": dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768,
                 beta_fast=32.0, beta_slow=1.0),
}
ROPE_BASE = 1e6


def _rotary_inputs(case, seed):
    g = _generator(seed)
    dtype = getattr(torch, case["dtype"])
    b, t, d = case["batch"], case["tokens"], case["dim"]
    q = _normal(g, b, t, case["q_heads"], d).to(dtype)
    k = _normal(g, b, t, case["kv_heads"], d).to(dtype)
    step = torch.randint(0, 3, (b, t), generator=g, device=DEV)  # tree depths repeat and skip
    return dict(q=q, k=k, positions=case["start"] + torch.cumsum(step, 1) // 2)


def _rules_inputs(case, seed):
    g = _generator(seed)
    n, vocab = case["rows"], case["vocab"]
    logits = (3.0 * _normal(g, n, vocab)).to(getattr(torch, case["dtype"]))
    # What was generated so far repeats itself: a skewed histogram.
    tokens = (vocab * torch.rand(case["seen"], generator=g, device=DEV) ** 3).long()
    counts = torch.zeros(vocab, dtype=torch.int32, device=DEV)
    counts.index_add_(0, tokens, torch.ones_like(tokens, dtype=torch.int32))
    depth = torch.randint(1, case["depth"] + 1, (n, 1), generator=g, device=DEV)
    paths = torch.randint(0, vocab, (n, case["depth"]), generator=g, device=DEV, dtype=torch.int32)
    # The tree's tokens are likely ones: each row's first is its best token.
    paths[:, 0] = logits.float().argmax(1).int()
    at = torch.arange(case["depth"], device=DEV)[None]
    paths = torch.where(at < depth, paths, torch.full_like(paths, -1))
    bias = 0.5 * _normal(g, vocab) if case["bias"] else None
    allowed = None
    if case["grammar"]:  # a few rows allow a handful of tokens, the last of many rows none
        words = (vocab + 31) // 32
        allowed = torch.randint(-2 ** 31, 2 ** 31, (n, words), generator=g, device=DEV).int()
        tight = torch.rand((n, 1), generator=g, device=DEV) < 0.3
        rare = torch.rand((n, words), generator=g, device=DEV) < 0.02
        allowed = torch.where(tight & ~rare, torch.zeros_like(allowed), allowed)
        if n > 4:
            allowed[n - 1] = 0
    return dict(logits=logits, counts=counts, paths=paths, bias=bias, allowed=allowed)


# -------------------------------------------------------------- plain forms --
def _plain_exponent(x, held):
    """The least e >= -60 with max |x| <= 127 2^e (int8) or 448 2^e (e4m3)
    over each block (the last two dimensions)."""
    m, e = torch.frexp(x.abs().amax(dim=(-2, -1)).float())
    if held == "int8":
        e = torch.where(m <= 127 / 128, e - 7, e - 6)
    else:
        e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(m == 0, MIN_EXPONENT, e).clamp_min(MIN_EXPONENT)


def _plain_fold(x, held):
    """x [B, H, n 64, D] -> codes [B, H, n, 64, D] and scales [B, H, n]."""
    b, h, t, d = x.shape
    x = x.reshape(b, h, t // BLOCK, BLOCK, d).float()
    scale = torch.ldexp(torch.ones((), device=x.device), _plain_exponent(x, held))
    y = x / scale[..., None, None]
    codes = y.round().to(torch.int8) if held == "int8" else y.to(torch.float8_e4m3fn)
    return codes, scale


def _plain_values(codes, scale):
    b, h, n, t, d = codes.shape
    return (codes.float() * scale[..., None, None]).view(b, h, n * t, d)


def _plain_attend(s):
    q, k_new, v_new, mask = s["q"].float(), s["k_new"].float(), s["v_new"].float(), s["mask"]
    k = torch.cat([_plain_values(*s["k8"]), s["k_tail"].float(), k_new], dim=2)
    v = torch.cat([_plain_values(*s["v8"]), s["v_tail"].float(), v_new], dim=2)
    b, hq, n, d = q.shape
    hk, keys = k.shape[1], k.shape[2]
    scores = (q.view(b * hk, hq // hk * n, d) @ k.view(b * hk, keys, d).transpose(1, 2).contiguous())
    scores = (scores * s["scale"]).view(b, hk, hq // hk, n, keys)
    if mask is None:
        at = torch.arange(keys, device=q.device)
        admit = (at[None] <= keys - n + torch.arange(n, device=q.device)[:, None])[None, None, None]
    else:
        admit = torch.ones(mask.shape[0], 1, 1, n, keys, dtype=torch.bool, device=q.device)
        admit[..., keys - mask.shape[-1]:] = mask[:, :, None]
    scores = torch.where(admit, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = p.view(b * hk, hq // hk * n, keys) @ v.view(b * hk, keys, d)
    out = out.view(b, hk, hq // hk, n, d) / torch.where(total == 0, 1.0, total)
    return out.view(b, hq, n, d).transpose(1, 2).to(torch.bfloat16).contiguous()


def _plain_fold_run(s):
    k, v, base, kept = s["k"], s["v"], s["base"], s["kept_index"]
    k = torch.cat([k[:, :, :base], k[:, :, base:][:, :, kept]], dim=2)
    v = torch.cat([v[:, :, :base], v[:, :, base:][:, :, kept]], dim=2)
    full = k.shape[2] // BLOCK * BLOCK
    k8, v8 = _plain_fold(k[:, :, :full], s["held"]), _plain_fold(v[:, :, :full], s["held"])
    k_read = torch.cat([_plain_values(*k8).to(torch.bfloat16), k[:, :, full:]], dim=2)
    v_read = torch.cat([_plain_values(*v8).to(torch.bfloat16), v[:, :, full:]], dim=2)
    return {"keys": k_read, "values": v_read, "scales": torch.stack([k8[1], v8[1]])}


def _plain_frequencies(case):
    """Radians per position of each pair, in 64 bits, and the factor that the
    stretched forms put on cos and sin."""
    rot, scaling = case["rotary"], SCALINGS[case["scaling"]]
    i = torch.arange(0, rot, 2, dtype=torch.float64, device=DEV)
    inv = ROPE_BASE ** (-i / rot)
    if scaling is None:
        return inv, 1.0
    factor = scaling["factor"]
    if scaling["rope_type"] == "linear":
        return inv / factor, 1.0
    old = scaling["original_max_position_embeddings"]
    if scaling["rope_type"] == "llama3":
        low, high = scaling["low_freq_factor"], scaling["high_freq_factor"]
        smooth = ((old * inv / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return (1 - smooth) * inv / factor + smooth * inv, 1.0
    first = rot * math.log(old / (scaling["beta_fast"] * 2 * math.pi)) / (2 * math.log(ROPE_BASE))
    last = rot * math.log(old / (scaling["beta_slow"] * 2 * math.pi)) / (2 * math.log(ROPE_BASE))
    first, last = max(math.floor(first), 0), min(math.ceil(last), rot - 1)
    ramp = ((torch.arange(rot // 2, dtype=torch.float64, device=DEV) - first)
            / max(last - first, 0.001)).clamp(0, 1)
    return inv / factor * ramp + inv * (1 - ramp), 0.1 * math.log(factor) + 1.0


def _plain_rotate(x, cos, sin, rot, interleaved):
    y = x.float()
    turned, rest = y[..., :rot], y[..., rot:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = turned[..., :rot // 2], turned[..., rot // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, rest], dim=-1).to(x.dtype).transpose(1, 2).contiguous()


def _plain_rotary(s):
    angle = s["positions"].double()[..., None] * s["frequencies"]
    cos = (torch.cos(angle) * s["factor"]).float()[:, :, None]
    sin = (torch.sin(angle) * s["factor"]).float()[:, :, None]
    return [_plain_rotate(s[x], cos, sin, s["rotary"], s["interleaved"]) for x in ("q", "k")]


def _plain_rules(s):
    x, paths, vocab = s["logits"].float(), s["paths"], s["logits"].shape[1]
    # Occurrences: of the whole sequence so far, and on each row's own path.
    onpath = torch.zeros((x.shape[0], vocab + 1), dtype=torch.int32, device=x.device)
    onpath.scatter_add_(1, torch.where(paths < 0, vocab, paths).long(), torch.ones_like(paths))
    count = s["counts"][None] + onpath[:, :vocab]
    y = torch.where(x < 0, x * s["repetition"], x / s["repetition"])
    y = y - (s["frequency"] * count + s["presence"])
    y = torch.where(count > 0, y, x)
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["allowed"] is not None:
        v = torch.arange(vocab, device=x.device)
        y = torch.where(((s["allowed"][:, v // 32] >> (v % 32)) & 1).bool(), y, -math.inf)
    if s["output"] == "logits":
        return y.to(s["logits"].dtype)
    best = y.amax(1, keepdim=True)
    first = torch.where(y == best, torch.arange(vocab, device=x.device), vocab).amin(1)
    return torch.where(best[:, 0] == -math.inf, -1, first)


# --------------------------------------------------------- prepare and run --
def prepare(case, seed):
    kind = case["kind"]
    if kind == "attend":
        s = _attend_inputs(case, seed)
        prefix = case["prefix"]
        full = prefix // BLOCK * BLOCK
        k, v = s.pop("k"), s.pop("v")
        s["k_new"], s["v_new"] = k[:, :, prefix:].contiguous(), v[:, :, prefix:].contiguous()
        if own:  # the cache a program has at this point of its sequence
            from specfit_amd.runtime import BlockKVCache
            cache = BlockKVCache(layers=1, kv_heads=case["kv_heads"], head_dim=case["dim"],
                                 capacity=prefix + case["new"], batch=case["batch"],
                                 tail_tokens=max(4096, case["new"]), held=case["held"], device=DEV)
            for at in range(0, prefix, 4096):
                to = min(prefix, at + 4096)
                cache.append(0, k[:, :, at:to], v[:, :, at:to])
                cache.commit()
            s["cache"], s["prefix"] = cache, prefix
        else:
            s["k8"] = _plain_fold(k[:, :, :full], case["held"])
            s["v8"] = _plain_fold(v[:, :, :full], case["held"])
            s["k_tail"], s["v_tail"] = (x[:, :, full:prefix].contiguous() for x in (k, v))
    elif kind == "fold":
        s = _fold_inputs(case, seed)
        s["held"] = case["held"]
        s["kept_index"] = torch.tensor(s["kept"], dtype=torch.long, device=DEV)
        if own:
            from specfit_amd.runtime import BlockKVCache
            s["cache"] = BlockKVCache(layers=1, kv_heads=case["kv_heads"], head_dim=case["dim"],
                                      capacity=case["tokens"], batch=case["batch"],
                                      tail_tokens=case["tokens"], held=case["held"], device=DEV)
    elif kind == "rotary":
        s = _rotary_inputs(case, seed)
        s["rotary"], s["interleaved"] = case["rotary"], case["interleaved"]
        if own:
            from specfit_amd.rotary import rotary_frequencies
            s["table"] = rotary_frequencies(case["dim"], base=ROPE_BASE, rotary_dim=case["rotary"],
                                            scaling=SCALINGS[case["scaling"]],
                                            interleaved=case["interleaved"], device=DEV)
        else:
            s["frequencies"], s["factor"] = _plain_frequencies(case)
    else:
        s = _rules_inputs(case, seed)
        s["output"] = case["output"]
        if own:
            from specfit_amd.runtime import LogitRules
            s["rules"] = LogitRules(counts=s["counts"], repetition=case["repetition"],
                                    presence=case["presence"], frequency=case["frequency"],
                                    bias=s["bias"])
        else:
            for name in ("repetition", "presence", "frequency"):
                s[name] = torch.tensor(case[name], dtype=torch.float32, device=DEV)
    s["kind"] = kind
    return s


def run(state):
    s, kind = state, state["kind"]
    if not own:
        return {"attend": _plain_attend, "fold": _plain_fold_run, "rotary": _plain_rotary,
                "rules": _plain_rules}[kind](s)
    if kind == "attend":
        cache = s["cache"]
        cache.append(0, s["k_new"], s["v_new"])
        out = cache.attend(0, s["q"], s["mask"], s["scale"])
        cache.crop(s["prefix"])  # the new tokens are not kept
        return out
    if kind == "fold":
        cache = s["cache"]
        cache.reset()
        cache.append(0, s["k"], s["v"])
        cache.compact(s["base"], s["kept"])
        cache.commit()
        keys, values = cache.read(0)
        return {"keys": keys, "values": values, "scales": cache.scales(0)}
    if kind == "rotary":
        from specfit_amd import ops
        return list(ops.rotary_embed(s["q"], s["k"], s["positions"], s["table"]))
    if s["output"] == "logits":
        return s["rules"].adjust(s["logits"], s["paths"], allowed=s["allowed"])
    return s["rules"].greedy(s["logits"], s["paths"], allowed=s["allowed"])


# ------------------------------------------------------------------- work --
def work(case):
    kind = case["kind"]
    if kind == "attend":
        b, hq, hk, d = case["batch"], case["q_heads"], case["kv_heads"], case["dim"]
        new, prefix = case["new"], case["prefix"]
        full = prefix // BLOCK * BLOCK
        cached = 2 * hk * (full * d + 4 * (full // BLOCK) + 2 * (prefix - full) * d)
        fresh = 2 * 2 * hk * new * d
        mask = {"causal": 0, "tree": new * new, "padded": b * new * (prefix + new)}[case["mask"]]
        pairs = new * prefix + (new * (new + 1) // 2 if case["mask"] == "causal" else new * new)
        return {"bytes": b * (cached + 2 * fresh + 2 * 2 * hq * new * d) + mask,
                "flops": 4 * b * hq * pairs * d}
    if kind == "fold":
        rows = 2 * case["batch"] * case["kv_heads"] * case["dim"]
        kept = case["tokens"] - case["tree"] + case["kept"]
        # Every row is read once and given back once in 16 bits, complete
        # blocks are written in 8.
        return {"bytes": rows * (2 * case["tokens"] + kept // BLOCK * BLOCK + 2 * kept),
                "flops": 2 * rows * kept}
    if kind == "rotary":
        size = 4 if case["dtype"] == "float32" else 2
        heads = case["batch"] * case["tokens"] * (case["q_heads"] + case["kv_heads"])
        return {"bytes": 2 * heads * case["dim"] * size + 8 * case["batch"] * case["tokens"],
                "flops": 3 * heads * case["rotary"]}
    n, vocab = case["rows"], case["vocab"]
    size = 4 if case["dtype"] == "float32" else 2
    moved = n * vocab * size * (2 if case["output"] == "logits" else 1) + 4 * vocab
    moved += 4 * n * case["depth"] + (4 * vocab if case["bias"] else 0)
    moved += n * ((vocab + 31) // 32) * 4 if case["grammar"] else 0
    return {"bytes": moved, "flops": 3 * n * vocab}


# ------------------------------------------------------------------ exact --
def _exact_held(x, held):
    """What a block cache gives back of x [B, H, T, D] (float64), and the
    scales of its complete blocks."""
    b, h, t, d = x.shape
    n = t // BLOCK
    blocks = x[:, :, :n * BLOCK].reshape(b, h, n, BLOCK * d)
    top = blocks.abs().amax(-1) if n else blocks.new_zeros((b, h, 0))
    limit = 127.0 if held == "int8" else 448.0
    guess = torch.ceil(torch.log2(torch.clamp(top, min=1e-300) / limit))
    for change in (1, -1):  # log2's rounding: the least power that holds the largest value
        other = guess + change
        if change == 1:
            guess = torch.where(top > limit * torch.exp2(guess), other, guess)
        else:
            guess = torch.where(top <= limit * torch.exp2(other), other, guess)
    scale = torch.exp2(torch.clamp(guess, min=float(MIN_EXPONENT)))
    y = blocks / scale[..., None]
    if held == "int8":
        y = torch.round(y)
    else:  # 3 bits after the leading one, steps no finer than 2^-9
        power = torch.floor(torch.log2(torch.clamp(y.abs(), min=2.0 ** -6)))
        power = torch.where(y.abs() < torch.exp2(power), power - 1, power)
        power = torch.where(y.abs() >= torch.exp2(power + 1), power + 1, power)
        step = torch.exp2(torch.clamp(power, min=-6.0) - 3)
        y = torch.round(y / step) * step
    y = (y * scale[..., None]).reshape(b, h, n * BLOCK, d)
    return torch.cat([y, x[:, :, n * BLOCK:]], dim=2), scale


def _exact_frequencies(case):
    scaling, rot = SCALINGS[case["scaling"]] or {"rope_type": "none"}, case["rotary"]
    form, found = scaling["rope_type"], []
    for pair in range(rot // 2):
        f = math.exp(-2 * pair / rot * math.log(ROPE_BASE))
        if form == "linear":
            f /= scaling["factor"]
        elif form == "llama3":
            # Turns over the original context decide how far a pair is slowed.
            turns = scaling["original_max_position_embeddings"] * f / (2 * math.pi)
            if turns < scaling["low_freq_factor"]:
                f /= scaling["factor"]
            elif turns < scaling["high_freq_factor"]:
                keep = ((turns - scaling["low_freq_factor"])
                        / (scaling["high_freq_factor"] - scaling["low_freq_factor"]))
                f *= keep + (1 - keep) / scaling["factor"]
        elif form == "yarn":
            # The pairs that make beta turns over the original context.
            at = [rot / 2 * math.log(scaling["original_max_position_embeddings"] / (2 * math.pi * beta))
                  / math.log(ROPE_BASE) for beta in (scaling["beta_fast"], scaling["beta_slow"])]
            first, last = max(0, math.floor(at[0])), min(rot - 1, math.ceil(at[1]))
            slow = min(1.0, max(0.0, (pair - first) / max(1e-3, last - first)))
            f *= 1 - slow + slow / scaling["factor"]
        found.append(f)
    factor = 1 + 0.1 * math.log(scaling["factor"]) if form == "yarn" else 1.0
    return torch.tensor(found, dtype=torch.float64, device=DEV), factor


def exact(case, seed):
    kind = case["kind"]
    if kind == "attend":
        s = _attend_inputs(case, seed)
        prefix, new, d = case["prefix"], case["new"], case["dim"]
        group = case["q_heads"] // case["kv_heads"]
        old_k, _ = _exact_held(s["k"][:, :, :prefix].double(), case["held"])
        old_v, _ = _exact_held(s["v"][:, :, :prefix].double(), case["held"])
        k = torch.cat([old_k, s["k"][:, :, prefix:].double()], dim=2)
        v = torch.cat([old_v, s["v"][:, :, prefix:].double()], dim=2)
        keys = prefix + new
        out = torch.zeros((case["batch"], new, case["q_heads"], d), dtype=torch.float64, device=DEV)
        for b in range(case["batch"]):
            if s["mask"] is None:
                admit = torch.ones((new, keys), dtype=torch.bool, device=DEV).tril(keys - new)
            else:
                m = s["mask"][b if s["mask"].shape[0] > 1 else 0, 0]
                admit = torch.ones((new, keys), dtype=torch.bool, device=DEV)
                admit[:, keys - m.shape[1]:] = m
            some = admit.any(1)
            for h in range(case["q_heads"]):
                a = s["q"][b, h].double() @ k[b, h // group].t() * s["scale"]
                p = torch.softmax(a.masked_fill(~admit, -math.inf), dim=-1)
                out[b, some, h] = p[some] @ v[b, h // group]
        return out
    if kind == "fold":
        s = _fold_inputs(case, seed)
        rows = list(range(s["base"])) + [s["base"] + p for p in s["kept"]]
        rows = torch.tensor(rows, dtype=torch.long, device=DEV)
        keys, sk = _exact_held(s["k"].index_select(2, rows).double(), case["held"])
        values, sv = _exact_held(s["v"].index_select(2, rows).double(), case["held"])
        return {"keys": keys, "values": values, "scales": torch.stack([sk, sv])}
    if kind == "rotary":
        s = _rotary_inputs(case, seed)
        rot, half = case["rotary"], case["rotary"] // 2
        inv, factor = _exact_frequencies(case)
        angle = s["positions"].double()[:, :, None] * inv
        turn = torch.polar(torch.full_like(angle, factor), angle)[:, :, None]
        out = []
        for x in (s["q"].double(), s["k"].double()):
            y = x.clone()
            if case["interleaved"]:
                z = torch.view_as_complex(x[..., :rot].reshape(*x.shape[:-1], half, 2).contiguous())
                y[..., :rot] = torch.view_as_real(z * turn).flatten(-2)
            else:
                z = torch.complex(x[..., :half].contiguous(), x[..., half:rot].contiguous()) * turn
                y[..., :rot] = torch.cat([z.real, z.imag], dim=-1)
            out.append(y.transpose(1, 2).contiguous())
        return out
    s = _rules_inputs(case, seed)
    single = lambda x: x.float().double()  # noqa: E731  each step of the definition rounds to 32 bits
    rep, pres, freq = (float(torch.tensor(case[n], dtype=torch.float32))
                       for n in ("repetition", "presence", "frequency"))
    result = []
    vocab = case["vocab"]
    for n in range(case["rows"]):
        x = s["logits"][n].double()
        count = s["counts"].double()
        path = s["paths"][n]
        count += torch.bincount(path[path >= 0].long(), minlength=vocab)
        y = single(torch.where(x < 0, x * rep, x / rep))
        y = single(y - single(single(freq * count) + pres))
        y = torch.where(count > 0, y, x)
        if s["bias"] is not None:
            y = single(y + s["bias"].double())
        if s["allowed"] is not None:
            bits = (s["allowed"][n][:, None] >> torch.arange(32, device=DEV)) & 1
            y = y.masked_fill(bits.flatten()[:vocab] == 0, -math.inf)
        if case["output"] == "logits":
            result.append(y)
        else:
            top = y.max()
            result.append(torch.nonzero(y == top)[0, 0] if top > -math.inf
                          else torch.tensor(-1, device=DEV))
    return torch.stack(result)
