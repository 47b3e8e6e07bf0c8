"""Which kernels the block attention's calls take: those that the GPU tests name for
theirs, so that a change of the rule cannot leave a kernel without a test."""
import pytest

from _block_forms import CASES, form_of
from specfit_amd import _native


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_the_form_of_a_call(case):
    assert form_of(case) == CASES[case]


def test_every_kernel_is_reached():
    """Staged and direct; unsplit, merged by rows and merged for many rows at once
    (2 to 16 splits of 512 rows and more over all heads); both head dims staged."""
    seen = set()
    for (B, Hq, _, D, Q, _), (rows, splits) in CASES.items():
        merge = "none" if splits == 1 else "many rows" if splits <= 16 and B * Hq * Q >= 512 else "rows"
        seen.add((rows, merge))
        seen.add((rows, D))
    assert seen >= {(rows, what) for rows in (16, 256)
                    for what in ("none", "rows", "many rows", 64, 128)}


def test_shapes_that_no_call_takes():
    rows = _native.lib().sf_block_attention_rows
    for args in ((0, 1, 64, 8, 2, 64), (1, 0, 64, 8, 2, 64), (1, 1, 0, 8, 2, 64),
                 (1, 1, 64, 9, 2, 64), (1, 1, 64, 8, 0, 64), (1, 1, 64, 8, 2, 96),
                 (1, 1, (1 << 30) + 1, 8, 2, 64), (1, 1 << 24, 64, 8, 2, 64)):
        assert rows(*args) == 0, args
