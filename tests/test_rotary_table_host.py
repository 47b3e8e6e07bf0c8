"""Rotary tables that the kernel could not read as it does: refused where they are
made, and anything else where it is used."""
from types import SimpleNamespace

import pytest
import torch

from specfit_amd import ops
from specfit_amd.rotary import RotaryTable, rotary_frequencies


@pytest.mark.parametrize("bad", [
    dict(turns=torch.zeros(32)), dict(turns=torch.zeros(31, dtype=torch.float64)),
    dict(turns=torch.zeros((2, 16), dtype=torch.float64)), dict(turns=torch.zeros(32).int()),
    dict(turns=torch.zeros(1, dtype=torch.float64).expand(32)),
    dict(turns=torch.zeros(64, dtype=torch.float64)[::2]), dict(rotary_dim=66), dict(rotary_dim=63),
    dict(rotary_dim=0, turns=torch.zeros(0, dtype=torch.float64)), dict(head_dim=32),
    dict(turns=[0.0] * 32)])
def test_tables_made_by_hand(bad):
    good = dict(head_dim=64, rotary_dim=64, interleaved=False, factor=1.0,
                turns=torch.zeros(32, dtype=torch.float64))
    RotaryTable(**good).to("cpu")
    with pytest.raises(ValueError):
        RotaryTable(**{**good, **bad})


def test_other_objects_are_no_tables():
    table = rotary_frequencies(64)
    other = SimpleNamespace(head_dim=64, rotary_dim=64, interleaved=False, factor=1.0,
                            turns=torch.zeros(32))
    q, positions = torch.zeros((1, 3, 2, 64)), torch.arange(3)
    with pytest.raises(TypeError, match="RotaryTable"):
        ops.rotary_embed(q, q, positions, other)
    with pytest.raises(ValueError, match="device"):  # a table: the next check
        ops.rotary_embed(q, q, positions, table)
