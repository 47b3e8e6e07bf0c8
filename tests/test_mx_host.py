"""Microscaled tensors and the refusals of their operators, without a GPU."""
import ctypes

import pytest
import torch

from specfit_amd import _native, mx, ops
from specfit_amd.mx import MXRows, MXWeight
from specfit_amd.runtime import Qwen3MXExperts

INVALID, UNSUPPORTED, MISALIGNED, TOO_MANY = 1, 2, 3, 4


def _bytes(seed, *shape):
    return torch.randint(0, 256, shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 31), (16, 32), (33, 100), (40, 512), (5, 1100)])
def test_weights_from_blocks_and_back(rows, dim):
    n = -(-dim // 32)
    codes, scales = _bytes(rows, rows, 16 * n), _bytes(dim, rows, n)
    w = MXWeight.from_blocks(codes, scales, dim)
    assert w.shape == (rows, dim) and w.codes.numel() == mx.weight_bytes(rows, dim)[0]
    back, back_scales = w.blocks()
    assert torch.equal(back_scales, scales)
    want = torch.stack([codes & 15, codes >> 4], -1).flatten(1)
    want[:, dim:] = 0                       # behind the rows' end
    assert torch.equal(torch.stack([back & 15, back >> 4], -1).flatten(1), want)
    # The place that the layout names for each value and scale.
    nibble = torch.stack([w.codes & 15, w.codes >> 4], -1).flatten()
    tiles, quads = -(-dim // 128), -(-dim // 512)
    for row, k in [(0, 0), (rows - 1, dim - 1), (rows // 2, dim // 3)]:
        tile, lane = k // 128, k % 128 // 32 * 16 + row % 16
        assert nibble[(((row // 16 * tiles + tile) * 64 + lane) * 16) * 2 + k % 32] == want[row, k]
        assert w.scales[((row // 16 * quads + tile // 4) * 64 + lane) * 4 + tile % 4] == scales[row, k // 32]


@pytest.mark.parametrize("dim", [1, 32, 130, 512, 1000])
def test_rows_hold_their_blocks(dim):
    code, scale = mx.row_bytes(dim)
    rows = MXRows(_bytes(1, 6 * code), _bytes(2, 6 * scale), (2, 3, dim), torch.bfloat16)
    assert rows.rows == 6 and rows.dim == dim and rows.device == torch.device("cpu")
    codes, scales = rows.blocks()
    assert torch.equal(codes, rows.codes.view(6, code)[:, :dim])
    for block in range(-(-dim // 32)):
        tile = block // 4
        at = tile // 4 * 16 + block % 4 * 4 + tile % 4
        assert torch.equal(scales[:, block], rows.scales.view(6, scale)[:, at])
    both = torch.cat([rows.codes, rows.scales])
    made = MXRows._of(both, (2, 3, dim), 6, torch.bfloat16)
    assert torch.equal(made.codes, rows.codes) and torch.equal(made.scales, rows.scales)
    assert made._pointers() == (made.codes.data_ptr(), made.scales.data_ptr())


def test_tensors_of_the_wrong_size_are_refused():
    code, scale = mx.row_bytes(100)
    good = _bytes(0, 2 * code), _bytes(0, 2 * scale)
    MXRows(*good, (2, 100), torch.bfloat16)
    for codes, scales, shape in [(good[0][1:], good[1], (2, 100)), (good[0], good[1][1:], (2, 100)),
                                 (*good, (3, 100)), (*good, (2, 0)), (*good, ()),
                                 (good[0].to(torch.int8), good[1], (2, 100)),
                                 (good[0].view(2, -1).t(), good[1], (2, 100))]:
        with pytest.raises(ValueError):
            MXRows(codes, scales, shape, torch.bfloat16)
    code, scale = mx.weight_bytes(20, 100)
    good = _bytes(0, code), _bytes(0, scale)
    MXWeight(*good, 20, 100)
    for args in [(good[0][1:], good[1], 20, 100), (good[0], good[1], 40, 100), (*good, 0, 100),
                 (*good, 20, 0), (good[0], good[1].float(), 20, 100)]:
        with pytest.raises(ValueError):
            MXWeight(*args)
    for codes, scales, dim in [(_bytes(0, 2, 48), _bytes(0, 2, 4), 100), (_bytes(0, 2, 64), _bytes(0, 2, 3), 100),
                               (_bytes(0, 64), _bytes(0, 4), 100), (_bytes(0, 0, 64), _bytes(0, 0, 4), 100),
                               (_bytes(0, 2, 64).float(), _bytes(0, 2, 4), 100), (_bytes(0, 2, 0), _bytes(0, 2, 0), 0)]:
        with pytest.raises(ValueError):
            MXWeight.from_blocks(codes, scales, dim)


def _weight(rows=32, dim=64):
    code, scale = mx.weight_bytes(rows, dim)
    return MXWeight(_bytes(0, code), _bytes(0, scale), rows, dim)


def _held(rows=2, dim=64, dtype=torch.bfloat16):
    code, scale = mx.row_bytes(dim)
    return MXRows(_bytes(0, rows * code), _bytes(0, rows * scale), (rows, dim), dtype)


def test_operators_refuse_what_they_cannot_do():
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16)
    plan = ops.DispatchPlan(2, 2, 4, torch.zeros((2, 5), dtype=torch.int32), torch.zeros(4, dtype=torch.int32),
                            torch.zeros(4, dtype=torch.int32))
    slots = torch.zeros((4, ops.mx_expert_bytes(64, 32)), dtype=torch.uint8)
    index = torch.zeros((2, 2), dtype=torch.int64)
    routes = torch.zeros((2, 2), dtype=torch.bfloat16)
    rows = torch.zeros((4, 64), dtype=torch.bfloat16)
    for call in [lambda: ops.mx_quantize(x), lambda: ops.mx_quantize_weight(x), lambda: ops.mx_values(_weight()),
                 lambda: ops.mx_values(_held()), lambda: ops.add_rms_norm(x, x, w, 1e-6),
                 lambda: ops.mx_linear(x, _weight()), lambda: ops.mx_linear(_held(), _weight()),
                 lambda: ops.mx_quantize_experts(torch.zeros((1, 3 * 64 * 32), dtype=torch.bfloat16), 64, 32),
                 lambda: ops.mx_grouped_swiglu(x, plan, None, slots, 64, 32, rows),
                 lambda: ops.mx_grouped_swiglu(_held(), plan, None, slots, 64, 32, rows),
                 lambda: ops.mx_routed_swiglu(x, index, routes, slots, 64, 32),
                 lambda: ops.mx_experts(x, index, routes, slots, 64, 32)]:
        with pytest.raises(ValueError, match="device"):     # there is no host form
            call()
    with pytest.raises(TypeError):
        ops.mx_linear(x, x)
    with pytest.raises(TypeError):
        ops.mx_values(x)
    with pytest.raises(TypeError):
        ops.mx_quantize(None)


def test_operators_refuse_inputs_that_want_gradients():
    x = torch.zeros((2, 64), requires_grad=True)
    plain, w = torch.zeros((2, 64)), torch.ones(64)
    plan = ops.DispatchPlan(2, 2, 4, *(torch.zeros(5, dtype=torch.int32) for _ in range(3)))
    for call in [lambda: ops.mx_quantize(x), lambda: ops.mx_quantize_weight(x),
                 lambda: ops.add_rms_norm(x, None, w, 1e-6), lambda: ops.add_rms_norm(plain, x, w, 1e-6),
                 lambda: ops.add_rms_norm(plain, None, x[0], 1e-6), lambda: ops.mx_linear(x, _weight()),
                 lambda: ops.mx_linear(_held(), _weight(), x[0]), lambda: ops.mx_quantize_experts(x, 64, 32),
                 lambda: ops.mx_grouped_swiglu(x, plan, None, x, 64, 32, x),
                 lambda: ops.mx_grouped_swiglu(_held(), plan, x, x, 64, 32, x),
                 lambda: ops.mx_routed_swiglu(x, plain, plain, plain, 64, 32),
                 lambda: ops.mx_routed_swiglu(_held(), plain, x, plain, 64, 32),
                 lambda: ops.mx_experts(x, plain, plain, plain, 64, 32),
                 lambda: ops.mx_experts(_held(), plain, x, plain, 64, 32)]:
        with pytest.raises(ValueError, match="no gradient"):
            call()


def test_modules_refuse_records_of_another_shape():
    nbytes = ops.mx_expert_bytes(64, 32)
    Qwen3MXExperts(torch.zeros((3, nbytes), dtype=torch.uint8), hidden_size=64, intermediate_size=32)
    for records in [torch.zeros((3, nbytes + 16), dtype=torch.uint8), torch.zeros((3, nbytes)),
                    torch.zeros((0, nbytes), dtype=torch.uint8), torch.zeros((257, nbytes), dtype=torch.uint8),
                    torch.zeros((3, 2 * nbytes), dtype=torch.uint8)[:, :nbytes]]:
        with pytest.raises(ValueError):
            Qwen3MXExperts(records, hidden_size=64, intermediate_size=32)
    module = Qwen3MXExperts(torch.zeros((3, nbytes), dtype=torch.uint8), hidden_size=64, intermediate_size=32)
    x, i, w = torch.zeros((2, 64), dtype=torch.bfloat16), torch.zeros((2, 2), dtype=torch.int64), torch.zeros((2, 2))
    for args in [(x[:, :32], i, w), (x[0], i, w), (x[:1], i, w), (x, i[0], w), (x, i, w[:, :1]), (x.float(), i, w)]:
        with pytest.raises(ValueError):
            module(*args)
    with pytest.raises(ValueError):
        ops.mx_expert_bytes(0, 32)


def test_records_are_the_three_weights_in_turn():
    lib = _native.lib()
    for hidden, inner in [(64, 32), (2048, 768), (33, 17), (1000, 424)]:
        at = (ctypes.c_int64 * 6)()
        assert lib.sf_mx_expert_parts(hidden, inner, at) == 0
        up, down = mx.weight_bytes(inner, hidden), mx.weight_bytes(hidden, inner)
        sizes = [up[0], up[0], down[0], up[1], up[1], down[1]]
        assert list(at) == [sum(sizes[:i]) for i in range(6)]
        assert lib.sf_mx_expert_bytes(hidden, inner) == sum(sizes)
        assert sum(sizes) % 16 == 0
    assert lib.sf_mx_expert_parts(64, 32, None) == INVALID


def test_the_library_refuses_before_any_launch():
    lib = _native.lib()
    a = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(a) + 63 & ~63          # 64-byte aligned, never read here
    q = lib.sf_mx_quantize
    assert q(0, None, 8, 0, 0, 8, 1, 0, None, 0, None, 0, None) == 0                # no rows
    assert q(0, None, 8, 0, 2, 8, 1, 0, p, 0, p, 0, None) == INVALID
    assert q(3, p, 8, 0, 2, 8, 1, 0, p, 0, p, 0, None) == INVALID                   # dtype
    assert q(0, p, 8, 0, 2, 8, 1, 2, p, 0, p, 0, None) == INVALID                   # held
    assert q(0, p, 8, 0, 2, 8, 3, 0, p, 0, p, 0, None) == INVALID                   # batch of rows
    assert q(0, p, -8, 0, 2, 8, 1, 0, p, 0, p, 0, None) == INVALID
    assert q(0, p, 8, 0, 2, (1 << 30) + 1, 1, 0, p, 0, p, 0, None) != 0
    assert q(0, p, 8, 0, 2, 8, 1, 0, p + 8, 0, p, 0, None) == q(0, p + 1, 8, 0, 2, 8, 1, 0, p, 0, p, 0, None) != 0
    misaligned = q(0, p + 1, 8, 0, 2, 8, 1, 0, p, 0, p, 0, None)
    unsupported = q(0, p, 8, 0, 2, (1 << 30) + 1, 1, 0, p, 0, p, 0, None)
    v = lib.sf_mx_values
    assert v(0, p, p, 0, 8, 0, p, None) == 0 and v(0, p, None, 2, 8, 0, p, None) == INVALID
    assert v(0, p + 4, p, 2, 8, 0, p, None) == v(0, p, p, 2, 8, 2, p + 2, None) == misaligned
    n = lib.sf_add_rms_norm
    assert n(0, p, 8, None, 0, 0, 8, p, 1e-6, None, p, None, None, None) == 0
    assert n(0, p, 8, None, 0, 2, 8, p, -1.0, None, p, None, None, None) == INVALID
    assert n(0, p, 8, None, 0, 2, 8, p, float("nan"), None, p, None, None, None) == INVALID
    assert n(0, p, 8, None, 0, 2, 8, p, 1e-6, p, p, None, None, None) == INVALID     # a sum of nothing
    assert n(0, p, 8, p, 8, 2, 8, p, 1e-6, None, None, None, None, None) == INVALID  # no output
    assert n(0, p, 8, p, 8, 2, 8, p, 1e-6, None, None, p, None, None) == INVALID     # codes without scales
    assert n(2, p + 2, 8, p, 8, 2, 8, p, 1e-6, p, p, p, p, None) == misaligned
    def lin(*args):                     # without a workspace
        return lib.sf_mx_linear(*args[:-1], None, args[-1])
    assert lin(3, p, p, 0, 0, 64, p, p, 32, None, 0, p, 32, None) == 0
    assert lin(2, p, p, 64, 2, 64, p, p, 32, None, 0, p, 32, None) == INVALID
    assert lin(3, p, None, 0, 2, 64, p, p, 32, None, 0, p, 32, None) == INVALID
    assert lin(3, p, p, 0, 2, 64, p, p, 32, None, 2, p, 32, None) == INVALID
    assert lin(3, p, p, 0, 2, 64, p, p, 32, None, 0, p, 31, None) == INVALID          # out stride
    assert lin(0, p, None, 64, 17, 64, p, p, 32, None, 0, p, 32, None) == unsupported  # 16 raw rows at most
    assert lin(0, p, None, 60, 2, 64, p, p, 32, None, 0, p, 32, None) == misaligned
    assert lin(0, p, None, 64, 2, 60, p, p, 32, None, 0, p, 32, None) == misaligned
    assert lin(3, p + 8, p, 0, 2, 64, p, p, 32, None, 0, p, 32, None) == misaligned
    assert lin(3, p, p, 0, 2, 64, p, p, 32, p + 1, 0, p, 32, None) == misaligned
    assert lib.sf_mx_linear(0, p, None, 64, 17, 64, p, p, 32, None, 0, p, 32, p + 8, None) == misaligned
    size = lib.sf_mx_linear_workspace
    assert size(3, 100, 64, 32) == size(0, 16, 64, 32) == size(1, 1, 2048, 16384) == 0
    assert size(0, 17, 100, 32) == 17 * sum(mx.row_bytes(100)) and size(1, 1, 2048, 16385) == sum(mx.row_bytes(2048))
    assert size(0, 1, 100, 32) == sum(mx.row_bytes(100)) and size(2, 1, 64, 32) == size(0, 1, 0, 32) == -1
    big = lib.sf_mx_expert_bytes(64, 32)
    g = lib.sf_mx_grouped_swiglu
    assert g(3, p, p, 0, p, p, None, 0, 2, 64, 32, 4, None, p, big, p, p, p, None) == 0
    assert g(3, p, p, 0, None, p, None, 2, 2, 64, 32, 4, None, p, big, p, p, p, None) == INVALID
    assert g(3, p, p, 0, p, p, None, 2, 2, 64, 32, 4, None, p, big - 16, p, p, p, None) == INVALID
    assert g(3, p, p, 0, p, p, None, 2, 2, 64, 32, 4, None, p, big + 8, p, p, p, None) == misaligned
    assert g(3, p, p, 0, p, p, None, 2, 2, 64, 32, 257, None, p, big, p, p, p, None) not in (0, INVALID, misaligned)
    assert g(0, p, None, 64, p, p, None, 17, 2, 64, 32, 4, None, p, big, p, p, p, None) == unsupported
    e = lib.sf_mx_experts
    assert e(0, p, None, 64, p, p, 0, 2, 64, 32, 4, p, big, p, p, None) == 0
    assert e(0, p, None, 64, p, p, 2, 2, 64, 32, 257, p, big, p, p, None) == INVALID
    assert e(0, p, None, 64, p, p, 2, 2, 64, 32, 4, p, big, None, p, None) == INVALID
    assert e(3, p, None, 0, p, p, 2, 2, 64, 32, 4, p, big, p, p, None) == INVALID
    assert e(1, p, None, 64, p, p, 2, 2, 64, 32, 4, p, big, p, p, None) == INVALID
    assert e(0, p, None, 64, p, p, 2, 2, 64, 32, 4, p, big, p + 4, p, None) == misaligned
    assert e(0, p, None, 64, p, p, 2, 2, 64, 32, 4, p, big - 16, p, p, None) == INVALID
    r = lib.sf_mx_routed_swiglu
    assert r(3, p, p, 0, p, p, 0, 2, 64, 32, 4, None, p, big, p, p, p, None) == 0
    assert r(3, p, p, 0, p, None, 2, 2, 64, 32, 4, None, p, big, p, p, p, None) == INVALID
    assert r(3, p, p, 0, p + 4, p, 2, 2, 64, 32, 4, None, p, big, p, p, p, None) == misaligned
    assert r(3, p, p, 0, p, p, 2, 0, 64, 32, 4, None, p, big, p, p, p, None) == INVALID


def test_few_routes_go_without_a_dispatch():
    form = _native.lib().sf_mx_experts_form
    assert form(1, 8, 2048, 768, 128) == form(8, 8, 2048, 768, 128) == form(1, 1, 64, 32, 1) == 1
    assert form(61, 8, 2048, 768, 128) == form(43, 3, 64, 32, 256) == form(4, 8, 4096, 1536, 8) == 0
    assert form(-1, 8, 2048, 768, 128) == form(1, 0, 64, 32, 4) == form(1, 1, 0, 32, 4) == -1


def test_the_workspace_holds_every_part():
    size = _native.lib().sf_mx_experts_workspace
    for tokens, top_k, hidden, inner, experts in [(1, 8, 2048, 768, 128), (500, 2, 33, 17, 6), (64, 8, 96, 300, 256)]:
        routes = tokens * top_k
        parts = [routes * sum(mx.row_bytes(inner)), tokens * sum(mx.row_bytes(hidden))]
        if not _native.lib().sf_mx_experts_form(tokens, top_k, hidden, inner, experts):
            parts += [8 * (experts + 1), 8 * routes, routes * (2 * hidden + -(-hidden // 32))]
        assert sum(parts) <= size(tokens, top_k, hidden, inner, experts) <= sum(parts) + 9 * 256
    assert size(1, 8, 64, 32, 257) == size(1, 8, 0, 32, 4) == size(1, 0, 64, 32, 4) == -1
    assert size(0, 2, 64, 32, 4) >= 0


def test_experts_are_refused_before_any_launch():
    """Calls whose rows are rounded first, with a dispatch and without, and calls
    whose routes are sorted first: without a GPU a launch would be an error of
    its own."""
    lib = _native.lib()
    a = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(a) + 63 & ~63
    big = lib.sf_mx_expert_bytes(64, 32)
    e = lib.sf_mx_experts
    for dtype, scales, stride, tokens, top_k, hidden, experts, dispatched in [
            (0, None, 64, 100, 2, 64, 4, True), (0, None, 63, 40, 2, 64, 4, False), (3, p, 0, 100, 2, 64, 4, True),
            (0, None, 64, 16, 16, 64, 4, True)]:
        assert lib.sf_mx_experts_form(tokens, top_k, hidden, 32, experts) == (not dispatched)
        def call(slots=p, slot=big, x=p, index=p, weights=p, stride=stride, workspace=p, out=p):
            return e(dtype, x, scales, stride, index, weights, tokens, top_k, hidden, 32, experts, slots, slot,
                     workspace, out, None)
        assert call(slot=big - 16) == INVALID and call(stride=-8) == INVALID
        for bad in [dict(slot=big + 8), dict(slots=p + 8), dict(index=p + 4), dict(weights=p + 1), dict(x=p + 1),
                    dict(workspace=p + 8), dict(out=p + 1)]:
            assert call(**bad) == MISALIGNED, bad
    # A grid of the second product or of the sum that does not fit.
    g = lib.sf_mx_grouped_swiglu
    wide = lib.sf_mx_expert_bytes(1 << 20, 32)
    assert g(3, p, p, 0, p, p, None, 1 << 23, 32, 1 << 20, 32, 4, None, p, wide, p, p, p, None) == UNSUPPORTED
    assert e(0, p, None, 1 << 20, p, p, 1 << 23, 32, 1 << 20, 32, 4, p, wide, p, p, None) == UNSUPPORTED


def test_workspaces_are_refused_for_shapes_that_the_calls_refuse():
    lib = _native.lib()
    a = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(a) + 63 & ~63
    size = lib.sf_mx_linear_workspace
    for rows, dim, out in [(1, 64, (1 << 28) + 1), ((1 << 20) + 1, 64, 64), (1, (1 << 24) + 1, 64),
                           (1 << 20, 32, 1 << 28)]:
        assert size(0, rows, dim, out) == size(3, rows, dim, out) == -1
        for dtype, stride in [(0, dim), (3, 0)]:
            assert lib.sf_mx_linear(dtype, p, p, stride, rows, dim, p, p, out, None, 0, p, out, p, None) == UNSUPPORTED
        with pytest.raises(ValueError):
            ops._mx_linear_workspace(0, rows, dim, out)
    assert size(0, 1 << 20, 1 << 24, 256) > 0 and size(3, 1, 64, 1 << 28) == 0
    size, big = lib.sf_mx_experts_workspace, lib.sf_mx_expert_bytes(64, 32)
    assert size(1 << 25, 8, 64, 32, 4) > 0
    assert size((1 << 25) + 1, 8, 64, 32, 4) == -1
    assert lib.sf_mx_experts(0, p, None, 64, p, p, (1 << 25) + 1, 8, 64, 32, 4, p, big, p, p, None) == INVALID
    with pytest.raises(ValueError):
        ops._mx_experts_workspace((1 << 25) + 1, 8, 64, 32, 4)


def test_the_limit_of_unrounded_rows_is_the_headers():
    import pathlib
    import re

    header = (pathlib.Path(ops.__file__).parent.parent / "include" / "specfit_amd.h").read_text()
    assert int(re.search(r"#define SF_MX_RAW_ROWS (\d+)", header)[1]) == ops._MX_RAW_ROWS
    size = _native.lib().sf_mx_linear_workspace
    assert size(0, ops._MX_RAW_ROWS, 64, 32) == 0 and size(0, ops._MX_RAW_ROWS + 1, 64, 32) > 0
