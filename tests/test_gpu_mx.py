"""Microscaled quantisation (K13), the norm with its 8-bit output (K14) and the
4-bit products (K15) against 64-bit references."""
import pytest
import torch

import _mx_reference as ref
from specfit_amd import ops
from specfit_amd.mx import MXWeight

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(seed, *shape):
    return torch.randn(shape, generator=_gen(seed), device=DEV)


def _spread(seed, rows, dim, dtype):
    """Values over many powers of two, zeros among them."""
    x = _normal(seed, rows, dim) * torch.exp2(6 * _normal(seed + 1, rows, dim))
    x = torch.where(_normal(seed + 2, rows, dim) > 1.5, 0.0, x)
    return x.clamp(-6e4, 6e4).to(dtype)


SIZES = [(1, 1), (1, 32), (3, 31), (2, 33), (17, 100), (16, 128), (5, 520), (33, 1000), (64, 2048),
         (2, 5000)]


# ------------------------------------------------------------------ K13 ----
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", SIZES)
def test_rows_to_e4m3(rows, dim, dtype):
    x = _spread(rows + dim, rows, dim, dtype)
    got = ops.mx_quantize(x)
    want, byte = ref.quantize(x, "e4m3")
    codes, scales = got.blocks()
    assert torch.equal(scales.long(), byte)
    assert torch.equal(got.values(torch.float32).double(), want)
    assert torch.equal(codes.view(torch.float8_e4m3fn).double()
                       * torch.exp2(byte.double() - 127).repeat_interleave(32, 1)[:, :dim], want)
    # What lies behind the rows' end is zeros.
    assert not got.codes.view(rows, -1)[:, dim:].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", SIZES)
def test_weight_to_e2m1(rows, dim, dtype):
    x = _spread(rows + dim, rows, dim, dtype)
    got = ops.mx_quantize_weight(x)
    want, byte = ref.quantize(x, "e2m1")
    codes, scales = got.blocks()
    assert torch.equal(scales.long(), byte)
    assert torch.equal(got.values(torch.float32).double(), want)
    four = torch.cat([ref.FOUR, -ref.FOUR]).to(DEV)
    pairs = torch.stack([codes & 15, codes >> 4], -1).flatten(1)[:, :dim]
    assert torch.equal(four[pairs.long()]
                       * torch.exp2(byte.double() - 127).repeat_interleave(32, 1)[:, :dim], want)
    again = MXWeight.from_blocks(codes, scales, dim)
    assert torch.equal(again.codes, got.codes)
    assert torch.equal(again.blocks()[1], scales)


@pytest.mark.parametrize("held", ["e4m3", "e2m1"])
def test_every_bf16_value_and_its_borders(held):
    """Each bf16 value in a block of its own and beside a large one."""
    every = torch.arange(65536, device=DEV, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = torch.zeros((65536, 64), dtype=torch.bfloat16, device=DEV)
    x[:, 0] = every
    x[:, 32] = 448.0
    x[:, 35] = every
    quantize = ops.mx_quantize if held == "e4m3" else ops.mx_quantize_weight
    got = quantize(x)
    want, byte = ref.quantize(x, held)
    assert torch.equal(got.blocks()[1].long(), byte)
    # fp32 has room for every product of a code and a scale but 2^128, to which
    # the largest bf16 values round: infinity there.
    got, want = got.values(torch.float32), want.float()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("held", ["e4m3", "e2m1"])
def test_non_finite_blocks_are_nan(held):
    x = _normal(0, 4, 100)
    x[0, 5], x[1, 40], x[2, 99] = float("nan"), float("inf"), float("-inf")
    q = (ops.mx_quantize if held == "e4m3" else ops.mx_quantize_weight)(x)
    bad = torch.zeros((4, 100), dtype=torch.bool, device=DEV)
    bad[0, :32] = bad[1, 32:64] = bad[2, 96:] = True
    assert torch.equal(torch.isnan(q.values()), bad)
    codes, scales = q.blocks()
    assert not codes[0, :16].any() and scales[0, 0] == 255


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_takes_any_strides(dtype):
    wide = _normal(3, 40, 300).to(dtype)
    views = [wide[:, 3:200], wide[::3], wide[:, ::2], wide.t(), wide[:, 8:264],
             wide[0].expand(7, 300), wide.view(4, 10, 300)[:, :, :33], wide.view(4, 10, 300)[1:, 2:5]]
    for v in views:
        assert torch.equal(ops.mx_quantize(v).values(), ops.mx_quantize(v.contiguous()).values())
        assert ops.mx_quantize(v).values().shape == v.shape
        if v.dim() == 2:
            assert torch.equal(ops.mx_quantize_weight(v).values(),
                               ops.mx_quantize_weight(v.contiguous()).values())


def test_values_in_each_type():
    x = _normal(4, 9, 77)
    for q in (ops.mx_quantize(x), ops.mx_quantize_weight(x)):
        for dtype in TYPES:
            assert torch.equal(q.values(dtype).double(), q.values(torch.float32).to(dtype).double())


def test_empty_inputs():
    assert ops.mx_quantize(torch.empty((0, 64), device=DEV)).values().shape == (0, 64)
    w = ops.mx_quantize_weight(_normal(0, 32, 64))
    x = torch.empty((2, 0, 64), dtype=torch.bfloat16, device=DEV)
    assert ops.mx_linear(x, w).shape == (2, 0, 32)
    total, y, q = ops.add_rms_norm(x, x, x.new_ones(64), 1e-6, quantized=True)
    assert total.shape == y.shape == q.values().shape == (2, 0, 64)


# ------------------------------------------------------------------ K14 ----
def _norm_reference(x, residual, weight, eps):
    s = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    r = (1 / torch.sqrt(s.double().square().mean(-1, keepdim=True) + eps)).float()
    return s, s.float() * r * weight.float()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 2048), (5, 64), (7, 100), (61, 520), (3, 1001),
                                      (4, 4096), (2, 5000), (3, 9000), (2, 20001), (300, 256), (2050, 800), (2100, 1001)])
def test_add_rms_norm(rows, dim, residual, dtype):
    x = _normal(rows, rows, dim).to(dtype)
    res = _normal(dim, rows, dim).to(dtype) * 3 if residual else None
    w = (1 + 0.3 * _normal(9, dim)).to(dtype)
    total, y, q = ops.add_rms_norm(x, res, w, 1e-6, quantized=True)
    s, want = _norm_reference(x, res, w, 1e-6)
    # The sum in fp32, rounded to the type: half a step, and half a fp32 step where
    # it has a longer tail than fp32 holds.
    assert residual or total is x
    assert (total.double() - (x.double() + (0 if res is None else res.double()))).abs().le(
        ref.half_step(s.double(), dtype) * 1.001).all()
    s, want = _norm_reference(total, None, w, 1e-6)
    # The same fp32 steps: equal, but where the mean's last bit moves r (never seen to).
    assert torch.equal(y, want.to(dtype))
    values, byte = ref.quantize(want, "e4m3")
    assert torch.equal(q.blocks()[1].long(), byte)
    assert torch.equal(q.values(torch.float32).double(), values)
    # Against 64 bits throughout: three fp32 roundings and the output's own.
    exact = total.double() / torch.sqrt(total.double().square().mean(-1, keepdim=True) + 1e-6) \
        * w.double()
    assert (y.double() - exact).abs().le(
        ref.half_step(exact, dtype) * (1 + 2.0 ** -8) + 4 * 2.0 ** -24 * exact.abs()).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_takes_any_strides_and_leaves_out_what_is_not_asked(dtype):
    wide, other = _normal(1, 30, 200).to(dtype), _normal(2, 30, 200).to(dtype)
    w = _normal(3, 96).to(dtype)
    for v, r in [(wide[:, 8:104], other[:, 16:112]), (wide[:, 3:99], other[:, :96]),
                 (wide[:, :192:2], other[:, 1:193:2]), (wide.view(5, 6, 200)[:, 1:4, :96],
                                                        other.view(5, 6, 200)[:, 2:5, 8:104])]:
        got = ops.add_rms_norm(v, r, w, 1e-5, quantized=True)
        want = ops.add_rms_norm(v.contiguous(), r.contiguous(), w, 1e-5, quantized=True)
        assert got[0].shape == got[1].shape == got[2].values().shape == v.shape
        for a, b in zip(got[:2], want[:2]):
            assert torch.equal(a, b)
        assert torch.equal(got[2].values(), want[2].values())
        only = ops.add_rms_norm(v, r, w, 1e-5, normed=False, quantized=True)
        assert only[1] is None and torch.equal(only[2].values(), want[2].values())
        plain = ops.add_rms_norm(v, None, w, 1e-5)
        assert plain[0] is v and plain[2] is None


def test_norm_of_extreme_rows():
    x = torch.zeros((4, 256), device=DEV)
    x[1] = 1e30            # squares beyond fp32
    x[2, 7] = float("inf")
    x[3] = 1e-30
    _, y, q = ops.add_rms_norm(x, None, torch.ones(256, device=DEV), 1e-6, quantized=True)
    assert not y[0].any() and not q.values()[0].any()
    assert torch.allclose(y[1], torch.ones(256, device=DEV), rtol=1e-6, atol=0)
    assert torch.isnan(y[2, 7]) and torch.isnan(q.values()[2, :32]).all()
    assert torch.allclose(y[3], torch.full((256,), 1e-27, device=DEV), rtol=1e-6, atol=0)
    _, y, _ = ops.add_rms_norm(x, None, torch.ones(256, device=DEV), 0.0)
    assert torch.isnan(y[0]).all()     # 0 / 0, as the formula has it


# ------------------------------------------------------------------ K15 ----
def _whole(seed, rows, dim, choices):
    pick = torch.randint(0, len(choices), (rows, dim), generator=_gen(seed), device=DEV)
    return torch.tensor(choices, device=DEV)[pick]


def _exact_case(seed, rows, dim, out, dtype):
    """Values whose products the matrix unit adds without loss: each eight's
    differ by less than 2^13, sums stay below 2^24 steps."""
    x = _whole(seed, rows, dim, [0.0, 1.0, -1.0, 2.0, -3.0, 4.0, 15.0, -14.0]).to(dtype)
    w = _whole(seed + 1, out, dim, [0.0, 0.5, -0.5, 1.0, 1.5, -2.0, 3.0, -4.0, 6.0, -6.0]).to(dtype)
    return x, w


LINEAR = [(1, 128, 16), (1, 2048, 5120), (2, 64, 24), (3, 40, 33), (16, 1000, 100), (17, 768, 2048),
          (32, 2048, 64), (33, 100, 47), (61, 2048, 1000), (64, 4096, 256), (100, 520, 330),
          (129, 128, 512), (255, 1024, 257), (256, 896, 512), (300, 136, 1030), (512, 2048, 768), (20, 64, 33000),
          (60, 200, 33000),
          (128, 64, 66000), (600, 640, 2500), (400, 96, 1100),
          (1000, 320, 96), (1, 8000, 48), (5, 2080, 4096), (2000, 1152, 4200), (16, 64, 70000),
          (7, 2048, 17000), (1600, 128, 9000), (4100, 72, 8000)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("held", [True, False])
@pytest.mark.parametrize("rows,dim,out", LINEAR)
def test_linear_places_every_value(rows, dim, out, held, dtype):
    x, w = _exact_case(rows + dim + out, rows, dim, out, dtype)
    q, weight = ops.mx_quantize(x), ops.mx_quantize_weight(w)
    assert torch.equal(q.values(dtype), x) and torch.equal(weight.values(dtype), w)
    bias = _whole(7, 1, out, [0.0, 3.0, -8.0])[0].to(dtype)
    want = x.double() @ w.double().t()
    assert torch.equal(ops.mx_linear(q if held else x, weight), want.to(dtype))
    assert torch.equal(ops.mx_linear(q if held else x, weight, bias), (want + bias.double()).to(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,dim,out", LINEAR)
def test_linear_against_64_bits(rows, dim, out, dtype):
    x = (_normal(rows, rows, dim) * torch.exp(_normal(2, rows, 1))).to(dtype)
    w = (0.05 * _normal(out, out, dim)).to(dtype)
    weight = ops.mx_quantize_weight(w)
    xv, wv = ref.quantize(x, "e4m3")[0], ref.quantize(w, "e2m1")[0]
    want = xv @ wv.t()
    for got in (ops.mx_linear(x, weight), ops.mx_linear(ops.mx_quantize(x), weight)):
        slack = ref.product_slack(xv[:64], wv)
        off = (got.double()[:64] - want[:64]).abs()
        assert off.le(slack + ref.half_step(want[:64], dtype) + slack * 2.0 ** -7).all()
        # Cut products err to either side: far below the bound on the whole.
        assert (got.double() - want).norm() <= 2.0 ** -8 * want.norm()


@pytest.mark.parametrize("rows", [1, 16, 17, 40, 200])
def test_scales_of_every_size_meet_their_blocks(rows):
    """One block in a row and in a weight row holds something: the product is
    theirs alone, whatever the scales."""
    dim, out = 1152, 96
    x = torch.zeros((rows, dim), device=DEV)
    w = torch.zeros((out, dim), device=DEV)
    g = _gen(rows)
    xb = torch.randint(0, dim // 32, (rows,), generator=g, device=DEV)
    for r in range(rows):
        x[r, 32 * int(xb[r]):][:32] = 2.0 ** (r % 20 - 10)
    for n in range(out):
        w[n, 32 * (n % (dim // 32)):][:32] = 2.0 ** (n % 13 - 6)
    x, w = x.to(torch.bfloat16), w.to(torch.bfloat16)
    got = ops.mx_linear(ops.mx_quantize(x), ops.mx_quantize_weight(w))
    assert torch.equal(got, (x.double() @ w.double().t()).to(torch.bfloat16))


@pytest.mark.parametrize("rows", [3, 20, 70, 300])
def test_nan_stays_in_its_row_and_column(rows):
    x = _normal(0, rows, 256).to(torch.bfloat16)
    w = _normal(1, 100, 256).to(torch.bfloat16)
    x[rows - 1, 200], w[7, 3] = float("nan"), float("inf")
    want = torch.zeros((rows, 100), dtype=torch.bool, device=DEV)
    want[rows - 1] = True
    want[:, 7] = True
    for held in (x, ops.mx_quantize(x)):
        assert torch.equal(torch.isnan(ops.mx_linear(held, ops.mx_quantize_weight(w))), want)


def test_linear_takes_strided_and_batched_rows():
    w = ops.mx_quantize_weight(_normal(0, 70, 96).to(torch.bfloat16))
    wide = _normal(1, 24, 400).to(torch.bfloat16)
    for v in (wide[:5, 8:104], wide[:5, 3:99], wide[:, :96], wide[:7, :192:2],
              wide.view(2, 12, 400)[:, 3:6, :96], wide.view(4, 6, 400)[..., 16:112], wide[0, :96]):
        got = ops.mx_linear(v, w)
        assert got.shape == (*v.shape[:-1], 70)
        assert torch.equal(got, ops.mx_linear(ops.mx_quantize(v.contiguous()), w))


def test_norm_then_products_as_a_layer_runs_them():
    """A residual stream through a norm and two products, the norm's rows
    straight into both."""
    rows, dim = 61, 2048
    h, o = (_normal(s, rows, dim).to(torch.bfloat16) for s in (1, 2))
    wn = (1 + 0.1 * _normal(3, dim)).to(torch.bfloat16)
    qkv, out = (ops.mx_quantize_weight(0.02 * _normal(s, n, dim)) for s, n in ((4, 640), (5, 2048)))
    total, y, q = ops.add_rms_norm(o, h, wn, 1e-6, quantized=True)
    a = ops.mx_linear(q, qkv)
    b = ops.mx_linear(q, out)
    total2, _, q2 = ops.add_rms_norm(b, total, wn, 1e-6, normed=False, quantized=True)
    xv = q.values(torch.float32).double()
    for got, w in ((a, qkv), (b, out)):
        want = xv @ w.values(torch.float32).double().t()
        assert (got.double() - want).norm() <= 2.0 ** -8 * want.norm()
    s = (b.double() + total.double()).to(torch.bfloat16)
    assert torch.equal(total2, s)
    assert torch.equal(q2.values(), ops.mx_quantize(_norm_reference(s, None, wn, 1e-6)[1]).values())


def test_weights_from_a_checkpoints_order():
    rows, dim = 50, 300
    g = _gen(0)
    codes = torch.randint(0, 256, (rows, 160), generator=g, device=DEV, dtype=torch.uint8)
    scales = torch.randint(120, 132, (rows, 10), generator=g, device=DEV, dtype=torch.uint8)
    w = MXWeight.from_blocks(codes, scales, dim)
    four = torch.cat([ref.FOUR, -ref.FOUR]).to(DEV)
    want = (four[torch.stack([codes & 15, codes >> 4], -1).flatten(1).long()]
            * torch.exp2(scales.double() - 127).repeat_interleave(32, 1))[:, :dim]
    assert torch.equal(w.values(torch.float32).double(), want)
    # One value of a row at a time picks one column of the weight.
    x = torch.eye(dim, dtype=torch.bfloat16, device=DEV)
    assert torch.equal(ops.mx_linear(x, w).double(), want.t())


def test_far_rows_and_outputs():
    """Offsets past 32 bits: what lies there equals what it is by itself."""
    rows, dim = 290_000, 8192
    x = torch.empty((rows, dim), dtype=torch.bfloat16, device=DEV).normal_(generator=_gen(1))
    w = (1 + 0.1 * _normal(2, dim)).to(torch.bfloat16)
    q = ops.mx_quantize(x)
    tail = x[-700:].clone()
    assert torch.equal(q.codes.view(rows, dim)[-700:], ops.mx_quantize(tail).codes.view(700, dim))
    values = q.values()
    assert torch.equal(values[-700:], ops.mx_quantize(tail).values())
    del values
    total, y, nq = ops.add_rms_norm(x, x, w, 1e-6, quantized=True)
    t2, y2, nq2 = ops.add_rms_norm(tail, tail, w, 1e-6, quantized=True)
    assert torch.equal(total[-700:], t2) and torch.equal(y[-700:], y2)
    assert torch.equal(nq.codes.view(rows, dim)[-700:], nq2.codes.view(700, dim))
    del total, y, nq
    weight = ops.mx_quantize_weight(x)              # 290,000 outputs
    assert torch.equal(weight.values()[-672:], ops.mx_quantize_weight(x[-672:]).values())
    out = ops.mx_linear(tail[:31], weight)
    assert torch.equal(out[:, -672:], ops.mx_linear(tail[:31], ops.mx_quantize_weight(x[-672:])))
    weight = ops.mx_quantize_weight(x[:8000])
    out = ops.mx_linear(q, weight)                  # 2.3e9 outputs
    # Whatever the tile, the same products are added in the same order.
    assert torch.equal(out[-600:], ops.mx_linear(x[-600:], weight))


def test_as_many_rows_as_a_product_takes():
    x = _normal(0, 1 << 20, 32).to(torch.bfloat16)
    w = ops.mx_quantize_weight(_normal(1, 24, 32))
    out = ops.mx_linear(x, w)
    assert torch.equal(out, ops.mx_linear(ops.mx_quantize(x), w))
    for part in (slice(0, 20000), slice(-20000, None)):
        assert torch.equal(out[part], ops.mx_linear(x[part], w))
    more = torch.cat([x, x[:1]])
    for rows in (more, ops.mx_quantize(more)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.mx_linear(rows, w)


def test_captured_chains_replay_each_their_own():
    """Two graphs of a layer's calls, replayed in turn, with eager work between."""
    rows, dim = 40, 512
    weights = [ops.mx_quantize_weight(0.05 * _normal(s, n, dim)) for s, n in ((1, 300), (2, dim))]
    wn = torch.ones(dim, dtype=torch.bfloat16, device=DEV)

    def chain(h, o):
        total, _, q = ops.add_rms_norm(o, h, wn, 1e-6, normed=False, quantized=True)
        return ops.mx_linear(q, weights[0]), ops.add_rms_norm(ops.mx_linear(total, weights[1]), total, wn, 1e-6)[1]

    inputs = [[_normal(s + i, rows, dim).to(torch.bfloat16) for i in range(2)] for s in (3, 5)]
    graphs, outs = [], []
    for h, o in inputs:
        chain(h, o)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(chain(h, o))
        graphs.append(graph)
    for step in range(4):
        for h, o in inputs:
            h.copy_(_normal(10 + step, rows, dim)), o.copy_(_normal(20 + step, rows, dim))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (h, o), out in zip(inputs, outs):
            want = chain(h, o)
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_each_operator_on_another_stream():
    rows, dim = 70, 384
    x = _normal(0, rows, dim).to(torch.bfloat16)
    wide = _normal(1, dim, rows).to(torch.bfloat16).t()     # copied to dense rows, on the stream
    w = torch.ones(dim, dtype=torch.bfloat16, device=DEV)
    want = (ops.mx_quantize(wide).values(), ops.mx_quantize_weight(wide).values(),
            *ops.add_rms_norm(x, wide, w, 1e-6)[:2], ops.mx_linear(wide, ops.mx_quantize_weight(x)))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    q, wq = ops.mx_quantize(wide, stream=side), ops.mx_quantize_weight(wide, stream=side)
    xw = ops.mx_quantize_weight(x, stream=side)
    got = (ops.mx_values(q, stream=side), ops.mx_values(wq, stream=side),
           *ops.add_rms_norm(x, wide, w, 1e-6, stream=side)[:2], ops.mx_linear(wide, xw, stream=side))
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,dim,out", [(1, 128, 16), (3, 40, 33), (20, 768, 520), (61, 520, 2048), (300, 136, 1030),
                                          (600, 640, 2500)])
def test_products_of_an_fp32_streams_rows(rows, dim, out, dtype):
    """Rows that a norm leaves of an fp32 stream, and rows of one 16-bit type with
    outputs of the other."""
    x, w = _exact_case(rows + dim + out, rows, dim, out, torch.float32)
    weight = ops.mx_quantize_weight(w)
    bias = _whole(7, 1, out, [0.0, 3.0, -8.0])[0].to(dtype)
    want = x.double() @ w.double().t()
    for held in (ops.mx_quantize(x), x.to(torch.bfloat16), x.to(torch.float16)):
        assert torch.equal(ops.mx_linear(held, weight, dtype=dtype), want.to(dtype))
        assert torch.equal(ops.mx_linear(held, weight, bias, dtype=dtype), (want + bias.double()).to(dtype))
    _, _, q = ops.add_rms_norm(x, _normal(1, rows, dim), _normal(2, dim), 1e-6, normed=False, quantized=True)
    got = ops.mx_linear(q, weight, dtype=dtype)
    assert got.dtype == dtype
    assert torch.equal(got, ops.mx_linear(ops.mx_quantize(q.values(dtype)), weight))


def test_products_refuse_outputs_in_other_types():
    x, weight = _normal(0, 4, 64), ops.mx_quantize_weight(_normal(1, 32, 64))
    rows = ops.mx_quantize(x)
    bias = torch.zeros(32, dtype=torch.bfloat16, device=DEV)
    for call in [lambda: ops.mx_linear(rows, weight), lambda: ops.mx_linear(rows, weight, dtype=torch.float32),
                 lambda: ops.mx_linear(x, weight), lambda: ops.mx_linear(x, weight, dtype=torch.bfloat16),
                 lambda: ops.mx_linear(rows, weight, bias, dtype=torch.float16),
                 lambda: ops.mx_linear(x.to(torch.bfloat16), weight, bias, dtype=torch.float16)]:
        with pytest.raises(ValueError):
            call()


def test_one_column_or_output_may_have_any_stride():
    """Of a dimension of one element torch gives any stride, and calls it contiguous."""
    w = _normal(0, 5, 7).to(torch.bfloat16)[:1, 3]
    b = _normal(1, 6, 9).to(torch.bfloat16)[2:3, 4]
    assert w.stride(0) != 1 and w.is_contiguous() and b.stride(0) != 1
    x = _normal(2, 40, 1).to(torch.bfloat16)
    for a, c in zip(ops.add_rms_norm(x, x, w, 1e-6)[:2], ops.add_rms_norm(x, x, w.clone(), 1e-6)[:2]):
        assert torch.equal(a, c)
    x, weight = _normal(3, 20, 64).to(torch.bfloat16), ops.mx_quantize_weight(_normal(4, 1, 64))
    assert torch.equal(ops.mx_linear(x, weight, b), ops.mx_linear(x, weight, b.clone()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,dim,out", [(1, 1, 1), (1, 7, 3), (40, 1, 1), (2, 1, 300), (17, 33, 1), (1000, 3, 2)])
def test_smallest_products(rows, dim, out, dtype):
    x, w = _exact_case(rows + dim + out, rows, dim, out, dtype)
    weight = ops.mx_quantize_weight(w)
    want = (x.double() @ w.double().t()).to(dtype)
    assert torch.equal(ops.mx_linear(x, weight), want)
    assert torch.equal(ops.mx_linear(ops.mx_quantize(x), weight), want)
