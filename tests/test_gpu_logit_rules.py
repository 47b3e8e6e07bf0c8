"""Rules on logits (K12) against their definition: every step is a
correctly rounded fp32 operation, so values and tokens are exact."""
import math

import pytest
import torch

from specfit_amd import ops
from specfit_amd.runtime import LogitRules

pytestmark = pytest.mark.gpu


def _single(x):
    return x.float().double()


def _reference(logits, counts, paths, rep, pres, freq, bias, allowed):
    """(y float64 holding fp32 values, tokens) of CPU tensors."""
    n, vocab = logits.shape
    x = logits.double()
    count = torch.zeros((n, vocab), dtype=torch.float64)
    if counts is not None:
        count += counts.double()
    if paths is not None:
        for r in range(n):
            row = paths[r][(paths[r] >= 0) & (paths[r] < vocab)].long()
            count[r] += torch.bincount(row, minlength=vocab)
    rep, pres, freq = (float(torch.tensor(v, dtype=torch.float32)) for v in (rep, pres, freq))
    y = _single(torch.where(x < 0, x * rep, x / rep))
    y = _single(y - _single(_single(freq * count) + pres))
    y = torch.where(count > 0, y, x)
    if bias is not None:
        y = _single(y + bias.double())
    if allowed is not None:
        bits = (allowed[..., None] >> torch.arange(32)) & 1
        bits = bits.flatten(-2)[..., :vocab].expand(n, vocab)
        y = torch.where(bits == 0, torch.full_like(y, -math.inf), y)
    key = torch.where(y.isnan(), torch.full_like(y, math.inf), y)
    best = key.amax(1, keepdim=True)
    nan = y.isnan()
    hit = torch.where(nan.any(1, keepdim=True), nan, y == best)
    tokens = torch.where(hit, torch.arange(vocab), vocab).amin(1)
    return y, torch.where(best[:, 0] == -math.inf, -1, tokens)


def _check(device, logits, *, counts=None, paths=None, rep=1.0, pres=0.0, freq=0.0, bias=None,
           allowed=None):
    y, tokens = _reference(logits, counts, paths, rep, pres, freq, bias, allowed)
    to = lambda t: None if t is None else t.to(device)  # noqa: E731
    args = dict(counts=to(counts), paths=to(paths), repetition=rep, presence=pres, frequency=freq,
                bias=to(bias), allowed=to(allowed))
    x = logits.to(device)
    before = x.clone()
    got = ops.adjust_logits(x, **args)
    assert torch.equal(torch.nan_to_num(x), torch.nan_to_num(before))
    assert got.dtype == logits.dtype
    want = y.float().to(logits.dtype)
    g = got.cpu()
    assert bool(((g == want) | (g.isnan() & want.isnan())).all())
    assert ops.greedy_tokens(x, **args).tolist() == tokens.tolist()
    ops.adjust_logits(x, out=x, **args)
    assert torch.equal(torch.nan_to_num(x), torch.nan_to_num(got))
    return y, tokens


def _words(g, n, vocab, share=0.5):
    words = (vocab + 31) // 32
    bits = torch.rand((n, words, 32), generator=g) < share
    value = (bits.long() << torch.arange(32)).sum(-1)
    return (value - (value >> 31 << 32)).int()  # as signed words


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32))
@pytest.mark.parametrize("n,vocab", [(1, 1), (3, 31), (2, 64), (5, 2048), (4, 2049), (9, 5000),
                                     (61, 32001), (2, 151936), (17, 4100)])
def test_all_rules(device, dtype, n, vocab):
    g = torch.Generator().manual_seed(n * vocab)
    logits = (3 * torch.randn((n, vocab), generator=g)).to(dtype)
    counts = torch.randint(0, 9, (vocab,), generator=g).int() * (torch.rand(vocab, generator=g) < 0.1)
    paths = torch.randint(-3, vocab + 2, (n, 9), generator=g).int()
    paths[:, 0] = logits.float().argmax(1)
    paths[:, 1] = paths[:, 0]  # the same token twice
    bias = torch.randn(vocab, generator=g)
    allowed = _words(g, n, vocab)
    allowed[-1] = 0
    rules = dict(counts=counts, paths=paths, rep=1.3, pres=0.25, freq=0.1)
    _check(device, logits, **rules)
    _check(device, logits, **rules, bias=bias)
    _check(device, logits, **rules, bias=torch.randn((n, vocab), generator=g), allowed=allowed)
    _, tokens = _check(device, logits, allowed=allowed)
    assert tokens[-1] == -1
    _check(device, logits, counts=counts, freq=0.7)
    _check(device, logits, paths=paths, pres=-1.0)
    _check(device, logits, allowed=allowed[0])
    _check(device, logits)


def test_ties_take_the_lowest_token(device):
    """Equal values in every place: across a thread's entries, wavefronts and
    workgroups, and equal only after a division."""
    for vocab in (70000, 70001):
        logits = torch.zeros((6, vocab))
        for r, at in enumerate(([5, 6], [300, 299], [2047, 2048], [69999, 513], [600, 65, 64000])):
            logits[r, at] = 4.0
        y, tokens = _check(device, logits)
        assert tokens.tolist() == [5, 299, 2047, 513, 65, 0]
        _check(device, logits.to(torch.bfloat16))
    logits = torch.zeros((1, 5000))
    logits[0, 4000], logits[0, 4500] = 16.5, 15.0  # 16.5 / 1.1 rounds to 15 in fp32
    y, tokens = _check(device, logits, paths=torch.tensor([[4000]], dtype=torch.int32), rep=1.1)
    assert y[0, 4000] == 15.0 and tokens.tolist() == [4000]


def test_values_that_are_not_finite(device):
    g = torch.Generator().manual_seed(1)
    logits = torch.randn((7, 3000), generator=g)
    logits[0, 50], logits[0, 60] = math.inf, math.nan      # a NaN is the largest
    logits[1] = -math.inf                                  # nothing to choose
    logits[2, 100] = math.inf
    logits[3, 7], logits[3, 2500] = math.nan, math.nan
    logits[4, 5] = -math.inf
    allowed = torch.full((7, 94), -1, dtype=torch.int32)
    _, tokens = _check(device, logits, allowed=allowed, counts=torch.ones(3000).int(), rep=1.5,
                       pres=0.5)
    assert tokens[0] == 60 and tokens[1] == -1 and tokens[2] == 100 and tokens[3] == 7
    allowed[:, 60 // 32] &= ~(1 << (60 % 32))              # what is not allowed has no effect
    _, tokens = _check(device, logits, allowed=allowed)
    assert tokens[0] == 50
    # Largest and least values, -0 beside 0.
    logits = torch.full((2, 100), -3.4028234e38)
    logits[1] = -0.0
    logits[1, 40] = 0.0
    _, tokens = _check(device, logits)
    assert tokens.tolist() == [0, 0]


@pytest.mark.parametrize("length", (0, 1, 64, 65, 200))
def test_paths_of_any_length(device, length):
    g = torch.Generator().manual_seed(length)
    logits = torch.randn((5, 4500), generator=g)
    paths = torch.randint(-1, 60, (5, length), generator=g).int()
    _check(device, logits, paths=paths, rep=1.2, freq=0.3)


def test_views(device):
    g = torch.Generator().manual_seed(2)
    wide = torch.randn((8, 5003), generator=g).to(device)
    counts = (torch.arange(5000) % 7 == 0).int().to(device)
    for x in (wide[:, :5000], wide[:, 3:5003], wide[::2, 1:5001], wide.T.contiguous().T[:, :5000],
              wide[:1, :5000].expand(4, -1)):
        got = ops.adjust_logits(x, counts=counts, repetition=1.5, presence=0.5)
        y, tokens = _reference(x.cpu(), counts.cpu(), None, 1.5, 0.5, 0.0, None, None)
        assert torch.equal(got.cpu(), y.float())
        assert ops.greedy_tokens(x, counts=counts, repetition=1.5, presence=0.5).tolist() == tokens.tolist()
    # Rows behind and between those written stay.
    out = torch.full((4, 5008), 7.0, device=device)
    ops.adjust_logits(wide[:4, :5000], counts=counts, repetition=1.5, out=out[:, 4:5004])
    assert bool((out[:, :4] == 7).all()) and bool((out[:, 5004:] == 7).all())
    bias = torch.randn((1, 5000), generator=g).to(device)
    a = ops.adjust_logits(wide[:, :5000], bias=bias)
    for b in (bias[0], bias.expand(8, -1)):
        assert torch.equal(ops.adjust_logits(wide[:, :5000], bias=b), a)


def test_rules_object(device):
    g = torch.Generator().manual_seed(3)
    rules = LogitRules.for_vocab(500, device, repetition=1.2, presence=0.1, frequency=0.2)
    tokens = torch.randint(0, 40, (3, 30), generator=g).to(device)
    rules.count(tokens)
    assert torch.equal(rules.counts.cpu(), torch.bincount(tokens.cpu().flatten(), minlength=500).int())
    logits = torch.randn((4, 500), generator=g).to(device)
    paths = torch.tensor([[1, -1], [2, 3], [2, 2], [499, -1]], dtype=torch.int32, device=device)
    y, best = _reference(logits.cpu(), rules.counts.cpu(), paths.cpu(), 1.2, 0.1, 0.2, None, None)
    assert torch.equal(rules.adjust(logits, paths).cpu(), y.float())
    assert rules.greedy(logits, paths).tolist() == best.tolist()
    with pytest.raises(ValueError, match="histogram"):
        LogitRules().count(tokens)


def test_captured_and_empty_calls(device):
    g = torch.Generator().manual_seed(4)
    logits = torch.randn((6, 3001), generator=g).to(device)
    rules = LogitRules.for_vocab(3001, device, repetition=1.5)
    rules.greedy(logits)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, adjusted = rules.greedy(logits), rules.adjust(logits)
    for turn in range(3):
        logits.copy_(torch.randn((6, 3001), generator=g))
        rules.count(torch.randint(0, 3001, (50,), generator=g).to(device))
        graph.replay()
        got = tokens.clone(), adjusted.clone()
        want = rules.greedy(logits), rules.adjust(logits)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert rules.greedy(logits[:0]).shape == (0,)
    assert rules.adjust(logits[:0]).shape == (0, 3001)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    other = ops.greedy_tokens(logits, counts=rules.counts, repetition=1.5, stream=stream)
    stream.synchronize()
    assert torch.equal(other, rules.greedy(logits))


def test_refusals(device):
    x = torch.zeros((2, 100), device=device)
    ints = lambda *s: torch.zeros(s, dtype=torch.int32, device=device)  # noqa: E731
    for args in (dict(counts=ints(99)), dict(counts=ints(100).long()), dict(counts=ints(100).cpu()),
                 dict(paths=ints(3, 4)), dict(paths=ints(2, 4).long()), dict(bias=x[0, :99]),
                 dict(bias=x[0].half()), dict(bias=torch.zeros((3, 100), device=device)),
                 dict(allowed=ints(3)), dict(allowed=ints(3, 4)), dict(allowed=ints(4).long()),
                 dict(repetition=0.0), dict(repetition=-1.0), dict(repetition=math.nan)):
        with pytest.raises(ValueError):
            ops.greedy_tokens(x, **args)
        with pytest.raises(ValueError):
            ops.adjust_logits(x, **args)
    for bad in (x.double(), x[0], x.cpu(), x[:, :0]):
        with pytest.raises(ValueError):
            ops.greedy_tokens(bad)
    for out in (x[:1], x.half(), x.cpu(), torch.zeros((2, 200), device=device)[:, ::2],
                torch.zeros((1, 100), device=device).expand(2, -1)):
        with pytest.raises(ValueError):
            ops.adjust_logits(x, out=out)


def test_another_stream_takes_its_own_copies(device):
    g = torch.Generator().manual_seed(9)
    x = torch.randn((3, 130), generator=g).to(device)
    paths = torch.randint(-1, 130, (3, 7), generator=g).int().to(device)
    bias = torch.randn((3, 130), generator=g).to(device)
    allowed = _words(g, 3, 130).to(device)
    args = dict(repetition=1.25, presence=0.5)
    want = ops.greedy_tokens(x, paths=paths, bias=bias, allowed=allowed, **args)
    turned = [t.t().contiguous().t() for t in (x, paths, bias, allowed)]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)
    got = ops.greedy_tokens(turned[0], paths=turned[1], bias=turned[2], allowed=turned[3],
                            stream=stream, **args)
    with torch.cuda.stream(stream):
        got = got.clone()
    stream.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_out_that_meets_an_argument_is_refused(device):
    room = torch.zeros((5, 64), device=device)
    ops.adjust_logits(room[:2], out=room[2:4])
    with pytest.raises(ValueError, match="share"):
        ops.adjust_logits(room[:2], out=room[1:3])
    with pytest.raises(ValueError, match="share"):
        ops.adjust_logits(room[:2], out=room[2:4], bias=room[3])
    with pytest.raises(ValueError, match="share"):
        ops.adjust_logits(room[:2], out=torch.as_strided(room, (2, 64), (128, 1)))
