"""Calls of the block attention that reach each of its kernels: the direct one (16
rows to a workgroup) and the staged one (256), with the keys in one piece or split,
and the splits merged by rows or, if few, for many rows at once.  Which shape takes
which is the library's choice; it is asked, so that a new rule moves the tests along."""
from specfit_amd import _native

# batch, query heads, KV heads, D, queries, keys
CASES = [
    # staged when this was written: 1 to 6 tiles in one piece, then 2 to 45 splits
    (3, 256, 1, 128, 17, 17), (8, 128, 2, 128, 17, 77), (5, 32, 1, 128, 130, 130),
    (8, 14, 2, 128, 200, 200), (5, 32, 4, 128, 130, 260), (2, 64, 1, 128, 200, 330),
    (5, 256, 1, 64, 17, 17), (8, 256, 1, 64, 17, 77), (2, 128, 2, 64, 130, 130),
    (3, 64, 1, 64, 200, 200), (3, 64, 4, 64, 200, 260), (2, 128, 2, 64, 200, 330),
    (5, 16, 4, 128, 333, 833), (8, 64, 4, 128, 17, 2017), (2, 64, 4, 128, 17, 6017),
    (3, 32, 1, 64, 300, 4300), (5, 32, 1, 64, 130, 4130), (1, 128, 2, 128, 17, 6017),
    (1, 64, 1, 128, 17, 20017), (1, 128, 2, 64, 17, 20017),
    # direct
    (2, 64, 4, 128, 9, 300), (1, 8, 2, 64, 1, 9001), (1, 32, 1, 128, 64, 2000),
]

MERGES = ("none", "rows", "many rows")
FORMS = [(rows, merge, D) for rows in (16, 256) for merge in MERGES for D in (64, 128)]


def splits_of(case):
    B, Hq, H, D, Q, S = case
    work = _native.lib().sf_block_attention_workspace(B, Q, S, Hq, H, D)
    splits, rest = divmod(work, B * Hq * Q * (D + 2) * 4)
    assert rest == 0
    return max(1, splits)


def form_of(case):
    """(rows of a workgroup, how splits are merged, head dim)."""
    B, Hq, H, D, Q, S = case
    splits = splits_of(case)
    merge = "none" if splits == 1 else "many rows" if splits <= 16 and B * Hq * Q >= 512 else "rows"
    return _native.lib().sf_block_attention_rows(B, Q, S, Hq, H, D), merge, D


def _one_of_each():
    """For every form the smallest of some thousand shapes that takes it."""
    best = {}
    grid = [(B, Hq, H, D, Q, Q + before) for B in (1, 2, 3, 5, 8)
            for Hq, H in ((8, 2), (32, 4), (64, 1), (14, 2), (128, 2)) for D in (64, 128)
            for Q in (1, 17, 64, 130, 300) for before in (0, 60, 500, 2000, 6000, 20000)]
    for case in grid:
        B, Hq, _, D, Q, S = case
        form, size = form_of(case), B * Hq * Q * S * D
        if form not in best or size < best[form][0]:
            best[form] = size, case
    return {form: case for form, (_, case) in best.items()}


ONE_OF_EACH = _one_of_each()
