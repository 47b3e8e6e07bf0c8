"""Rotary positions (K11) against the formula in 64 bits.

A turned element is two products and a sum of fp32 values: with sines good to
2^-22 (their own rounding, that of the reduced angle, 2^-25 of a turn at most, and
that of the factor), it is off by at most (|a| + |b|) (2^-22 + 3 2^-24) factor, and
by half a step of its type."""
import math

import pytest
import torch

from _block_reference import EPS
from specfit_amd import ops
from specfit_amd.rotary import RotaryTable, rotary_frequencies

pytestmark = pytest.mark.gpu


def _reference(x, positions, table):
    """x [B, T, H, D] (any float type, CPU) -> ([B, H, T, D] float64, bound)."""
    y = x.double()
    rot = table.rotary_dim
    angle = positions.double()[..., None] * table.turns.cpu()
    angle = (angle - angle.round()) * 2 * math.pi
    cos, sin = (f(angle)[:, :, None] * table.factor for f in (torch.cos, torch.sin))
    if table.interleaved:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        size = (a.abs() + b.abs()).repeat_interleave(2, -1)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        size = (a.abs() + b.abs()).repeat(1, 1, 1, 2)
    out = torch.cat([turned, y[..., rot:]], -1)
    bound = torch.zeros_like(out)
    # + the smallest step of the type: results below its normal range.
    bound[..., :rot] = size * (2.0 ** -22 + 3 * 2.0 ** -24) * table.factor \
        + EPS[x.dtype] * turned.abs() * (1 + 2.0 ** -20) + torch.finfo(x.dtype).tiny * EPS[x.dtype] * 2
    return out.transpose(1, 2), bound.transpose(1, 2)


def _check(q, k, positions, table):
    got = ops.rotary_embed(q, k, positions, table)
    where = positions.cpu()
    where = (where[None] if where.dim() == 1 else where).expand(q.shape[0], -1)
    for x, y in zip((q, k), got):
        want, bound = _reference(x.cpu(), where, table)
        assert y.dtype == x.dtype and y.shape == want.shape and y.is_contiguous()
        err = (y.cpu().double() - want).abs()
        assert bool((err <= bound).all()), (err - bound).max().item()
    return got


def _rand(g, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g).to(dtype)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32))
@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("B,T,Hq,Hk,D,rot", [
    (1, 1, 32, 4, 128, 128), (1, 61, 32, 4, 128, 128), (2, 7, 8, 8, 64, 32), (3, 33, 5, 1, 80, 80),
    (1, 5, 3, 2, 96, 24), (2, 9, 2, 1, 50, 18), (1, 2, 2, 2, 7, 6), (1, 1200, 4, 2, 256, 256),
    (1, 3, 1, 1, 1024, 1024), (2, 2500, 2, 1, 64, 64)])
def test_layouts_and_sizes(device, dtype, interleaved, B, T, Hq, Hk, D, rot):
    g = torch.Generator().manual_seed(T + D)
    table = rotary_frequencies(D, base=1e6, rotary_dim=rot, interleaved=interleaved, device=device)
    q, k = (_rand(g, B, T, h, D, dtype=dtype).to(device) for h in (Hq, Hk))
    positions = torch.randint(0, 40960, (B, T), generator=g).to(device)
    got = _check(q, k, positions, table)
    if rot < D:
        assert torch.equal(got[0][..., rot:], q.transpose(1, 2)[..., rot:])


@pytest.mark.parametrize("scaling", [
    dict(rope_type="linear", factor=4.0), dict(rope_type="dynamic", factor=2.0),
    dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
         original_max_position_embeddings=8192),
    dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768)])
def test_scaled_forms(device, scaling):
    g = torch.Generator().manual_seed(3)
    table = rotary_frequencies(128, base=1e6, scaling=scaling, max_position_embeddings=32768,
                               seq_len=100000, device=device)
    q, k = (_rand(g, 2, 40, h, 128, dtype=torch.float32).to(device) for h in (4, 2))
    _check(q, k, torch.randint(0, 131072, (2, 40), generator=g).to(device), table)


def test_far_and_negative_positions(device):
    """Positions from -10^9 to 2^40 keep their angles: the bound is that of
    small positions but for the fp64 product (2^-53 of up to 2^38 turns)."""
    g = torch.Generator().manual_seed(4)
    table = rotary_frequencies(64, base=10000.0, device=device)
    q, k = (_rand(g, 1, 9, h, 64, dtype=torch.float32).to(device) for h in (3, 1))
    for positions in ([0, 1, -1, 10 ** 6, 10 ** 6 + 1, -10 ** 9, 2 ** 31, 2 ** 31 - 1, 2 ** 33],):
        _check(q, k, torch.tensor(positions, device=device), table)
    far = torch.full((9,), 2 ** 40, device=device)
    _check(q, k, far, table)


def test_positions_of_every_shape(device):
    g = torch.Generator().manual_seed(5)
    table = rotary_frequencies(64, device=device)
    q, k = (_rand(g, 3, 6, h, 64).to(device) for h in (2, 1))
    row = torch.arange(6, device=device) * 7
    a = ops.rotary_embed(q, k, row, table)
    for positions in (row[None], row.expand(3, 6), row.repeat(3, 2)[:, :6],
                      torch.stack([row] * 3, 1).T):
        b = ops.rotary_embed(q, k, positions, table)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_views(device):
    """Heads out of a fused projection, transposed, at odd offsets, strided."""
    g = torch.Generator().manual_seed(6)
    table = rotary_frequencies(64, rotary_dim=48, device=device)
    positions = torch.arange(10, device=device)[None]
    fused = _rand(g, 2, 10, 6 * 64).to(device)
    cases = [(fused[..., :256].view(2, 10, 4, 64), fused[..., 256:].view(2, 10, 2, 64)),
             tuple(_rand(g, 2, h, 10, 64).to(device).transpose(1, 2) for h in (4, 2)),
             tuple(_rand(g, 2, 10, h, 67).to(device)[..., 3:] for h in (4, 2)),
             tuple(_rand(g, 2, 10, h, 128).to(device)[..., ::2] for h in (4, 2)),
             (_rand(g, 1, 10, 4, 64).to(device).expand(2, -1, -1, -1),
              _rand(g, 2, 10, 1, 64).to(device).expand(-1, -1, 2, -1))]
    for q, k in cases:
        _check(q, k, positions.expand(2, -1), table)


def test_against_the_bf16_table_of_a_model(device):
    """Near positions agree with transformers' cosines to bf16's steps."""
    from transformers import Qwen3MoeConfig
    from transformers.models.qwen3_moe.modeling_qwen3_moe import (Qwen3MoeRotaryEmbedding,
                                                                    apply_rotary_pos_emb)
    config = Qwen3MoeConfig(num_attention_heads=4, num_key_value_heads=2, head_dim=128,
                            hidden_size=64, max_position_embeddings=40960,
                            rope_parameters={"rope_type": "default", "rope_theta": 1e6})
    table = RotaryTable.from_config(config, device=device)
    g = torch.Generator().manual_seed(7)
    q, k = (_rand(g, 1, 50, h, 128, dtype=torch.float32).to(device) for h in (4, 2))
    positions = torch.arange(50, device=device)[None]
    cos, sin = Qwen3MoeRotaryEmbedding(config).to(device)(q, positions)
    want = apply_rotary_pos_emb(q.transpose(1, 2), k.transpose(1, 2), cos, sin)
    for x, y in zip(ops.rotary_embed(q, k, positions, table), want):
        # fp32 angles of up to 50 radians: 50 2^-23 each, on |a| + |b| < 10.
        assert (x - y).abs().max().item() < 50 * 2.0 ** -23 * 10


def test_captured_and_empty_calls(device):
    g = torch.Generator().manual_seed(8)
    table = rotary_frequencies(64, device=device)
    q, k = (_rand(g, 1, 4, h, 64).to(device) for h in (4, 2))
    positions = torch.arange(4, device=device)
    ops.rotary_embed(q, k, positions, table)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.rotary_embed(q, k, positions, table)
    for turn in range(3):
        q.copy_(_rand(g, 1, 4, 4, 64).to(device))
        positions.add_(100)
        graph.replay()
        got = [t.clone() for t in out]
        want = ops.rotary_embed(q, k, positions, table)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    empty = ops.rotary_embed(q[:, :0], k[:, :0], positions[:0], table)
    assert empty[0].shape == (1, 4, 0, 64)
    one = ops.rotary_embed(q, k[:, :, :0], positions, table)
    assert one[1].shape == (1, 0, 4, 64) and torch.equal(one[0], ops.rotary_embed(q, k, positions, table)[0])


def test_refusals(device):
    table = rotary_frequencies(64, device=device)
    q = torch.zeros((1, 3, 2, 64), dtype=torch.bfloat16, device=device)
    positions = torch.arange(3, device=device)
    with pytest.raises(ValueError, match="bf16"):
        ops.rotary_embed(q.double(), q.double(), positions, table)
    with pytest.raises(ValueError, match="dtype"):
        ops.rotary_embed(q, q.half(), positions, table)
    with pytest.raises(ValueError, match="dtype"):
        ops.rotary_embed(q, q, positions.int(), table)
    with pytest.raises(ValueError, match="same tokens"):
        ops.rotary_embed(q, q[:, :2], positions, table)
    with pytest.raises(ValueError, match="positions"):
        ops.rotary_embed(q, q, torch.arange(4, device=device), table)
    with pytest.raises(ValueError, match="head dim"):
        ops.rotary_embed(q[..., :32], q[..., :32], positions, table)
    with pytest.raises(ValueError, match="share a device"):
        ops.rotary_embed(q, q, positions, table.to("cpu"))
    with pytest.raises(ValueError, match="HIP device"):
        ops.rotary_embed(q.cpu(), q.cpu(), positions.cpu(), table)


def test_another_stream_takes_its_own_copies(device):
    g = torch.Generator().manual_seed(8)
    table = rotary_frequencies(64, device=device)
    q, k = (torch.randn((1, 5, h, 64), generator=g).to(device) for h in (4, 2))
    positions = torch.tensor([[3, 0], [9, 0], [7, 0], [5, 0], [1, 0]], device=device)[:, 0]
    want = ops.rotary_embed(q, k, positions, table)
    views = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k)]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)
    got = ops.rotary_embed(*views, positions, table, stream=stream)
    with torch.cuda.stream(stream):
        copies = [t.clone() for t in got]
    stream.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(copies[0], want[0]) and torch.equal(copies[1], want[1])
