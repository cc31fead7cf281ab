"""Attention of rows that share pages where the plan has tiles of what they share: every test looks for
such items in the plan's words (flag 2) before it compares the context with the plain 64-bit form."""
import pytest
import torch

import paged_ref as pr
from test_paged_gpu import covered, decode
from test_ranges_gpu import close

pytestmark = pytest.mark.gpu


def tiles(plan, nseq):
    """(first row, rows) of the plan's items over shared blocks."""
    d = plan.data.cpu().tolist()
    at = (16 + 12 * nseq + 15) // 16 * 16
    items = [d[at + 16 * i:at + 16 * i + 16] for i in range(d[0])]
    return [(e[0], e[1]) for e in items if e[3] & 2]


@pytest.mark.parametrize("shape", [(4, 4, 64), (8, 2, 128), (12, 1, 64), (16, 1, 128), (6, 2, 64)], ids=str)
@pytest.mark.parametrize("own", [0, 37])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_bias_of_a_tile_of_one_row(gpu, shape, own, cap):
    """A group of one row more than a tile holds, scores biased by distance: the last row is a tile of its own. With
    positions behind the prefix, and with none."""
    per = 32 // (shape[0] // shape[1])
    n = per + 1
    lengths = [832 + (own + 3 * t if own else 0) for t in range(n)]
    laid = pr.Laid(lengths, shape[1], shape[2], 64, [0, n], [832], seed=3)
    got, want, tol, plan = decode(gpu, laid, shape, lengths, list(range(n)), [0, n], [832], softcap=cap, bias=True)
    assert (per, 1) in tiles(plan, n)
    close(got, want, tol)


@pytest.mark.parametrize("shape,n,doc", [((24, 8, 64), 500, 0), ((48, 16, 64), 250, 0), ((24, 8, 64), 300, 704),
                                         ((3, 1, 128), 800, 704)], ids=str)
def test_pairs_of_rows(gpu, shape, n, doc):
    """Two rows of each of many sequences, three query heads a kv head: five such pairs in a tile's ten rows. Every block
    that a row sees is in one item of its own, and every row's context is its own."""
    lens = [doc + 2 + 7 * t % 80 for t in range(n)]
    laid = pr.Laid(lens, shape[1], shape[2], 32, [0, n], [doc], seed=3, cols=24 + 3)
    tk = [m - 1 + j for m in lens for j in range(2)]
    row = [t for t in range(n) for _ in range(2)]
    got, want, tol, plan = decode(gpu, laid, shape, tk, row, [0, 2 * n] if doc else None, [doc] if doc else None, max_tk=800)
    for r, blocks in enumerate(covered(plan, 2 * n, 3)):
        assert sorted(blocks) == list(range((lens[row[r]] + 31) // 32)), r  # the pair's
    assert bool(tiles(plan, 2 * n)) == bool(doc)
    close(got, want, tol)
