"""Which kernels the block attention's calls take: the GPU tests have shapes for all
of them."""
from _block_forms import CASES, FORMS, ONE_OF_EACH, form_of
from specfit_amd import _native


def test_every_kernel_is_reached():
    """A form that no shape takes any more would be code without a call."""
    assert set(ONE_OF_EACH) == set(FORMS)
    assert all(form_of(case) == form for form, case in ONE_OF_EACH.items())
    assert {form_of(case)[0] for case in CASES} == {16, 256}


def test_shapes_that_no_call_takes():
    rows = _native.lib().sf_block_attention_rows
    for args in ((0, 1, 64, 8, 2, 64), (1, 0, 64, 8, 2, 64), (1, 1, 0, 8, 2, 64),
                 (1, 1, 64, 9, 2, 64), (1, 1, 64, 8, 0, 64), (1, 1, 64, 8, 2, 96),
                 (1, 1, (1 << 30) + 1, 8, 2, 64), (1, 1 << 24, 64, 8, 2, 64)):
        assert rows(*args) == 0, args
