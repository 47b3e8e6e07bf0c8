"""Calls of the block attention that reach each of its kernels: the direct one (16
rows to a workgroup) and the staged one (256), unsplit or with the keys split and
merged by rows (many splits or few rows) or by many rows at once."""
from specfit_amd import _native

# batch, query heads, KV heads, D, queries, keys: rows of a workgroup, splits
CASES = {
    (3, 256, 1, 128, 17, 17): (256, 1), (8, 128, 2, 128, 17, 77): (256, 1),  # 1 tile, 2 tiles
    (5, 32, 1, 128, 130, 130): (256, 1), (8, 14, 2, 128, 200, 200): (256, 1),
    (5, 32, 4, 128, 130, 260): (256, 1), (2, 64, 1, 128, 200, 330): (256, 1),
    (5, 256, 1, 64, 17, 17): (256, 1), (8, 256, 1, 64, 17, 77): (256, 1),
    (2, 128, 2, 64, 130, 130): (256, 1), (3, 64, 1, 64, 200, 200): (256, 1),
    (3, 64, 4, 64, 200, 260): (256, 1), (2, 128, 2, 64, 200, 330): (256, 1),
    (5, 16, 4, 128, 333, 833): (256, 2), (8, 64, 4, 128, 17, 2017): (256, 4),
    (2, 64, 4, 128, 17, 6017): (256, 16), (3, 32, 1, 64, 300, 4300): (256, 2),
    (5, 32, 1, 64, 130, 4130): (256, 3), (1, 128, 2, 128, 17, 6017): (256, 24),
    (1, 64, 1, 128, 17, 20017): (256, 45), (1, 128, 2, 64, 17, 20017): (256, 23),
    (2, 64, 4, 128, 9, 300): (16, 1), (1, 8, 2, 64, 1, 9001): (16, 18),
    (1, 32, 1, 128, 64, 2000): (16, 2),
}


def form_of(case):
    """(rows of a workgroup, splits) of a call."""
    B, Hq, H, D, Q, S = case
    lib = _native.lib()
    work = lib.sf_block_attention_workspace(B, Q, S, Hq, H, D)
    splits, rest = divmod(work, B * Hq * Q * (D + 2) * 4)
    assert rest == 0
    return lib.sf_block_attention_rows(B, Q, S, Hq, H, D), max(1, splits)
