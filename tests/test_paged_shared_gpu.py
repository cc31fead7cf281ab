"""Attention of rows that share pages where the plan has tiles of what they share: every test looks for
such items in the plan's words (flag 2) before it compares the context with the plain 64-bit form."""
import math
import random

import pytest
import torch

import paged_ref as pr
from test_paged_gpu import covered, decode, ints, put, queries
from test_ranges_gpu import close, slopes_of

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


# lengths, (heads, kv, hd), page, groups' first rows, prefixes, window, shared, softcap, bias, rows of the shared tiles
FORMS = [
    ([830, 829, 768], (8, 2, 128), 64, [0, 3], [768], 0, 0, 0.0, False, {(0, 3)}),
    ([730, 800], (32, 8, 128), 32, [0, 2], [704], 0, 0, 0.0, True, {(0, 2)}),
    ([900, 901, 902, 903, 904, 1100, 905, 906, 896], (8, 2, 128), 128, [0, 9], [896], 0, 0, 50.0, True, {(0, 8), (8, 1)}),
    ([900] * 33 + [17], (4, 4, 64), 32, [0, 33], [864], 0, 0, 0.0, False, {(0, 32), (32, 1)}),
    ([700, 650, 130, 664, 664, 900, 910], (16, 1, 128), 64, [0, 2, 3, 5, 7], [640, 128, 640, 832], 0, 0, 30.0, True,
     {(0, 2), (3, 2), (5, 2)}),
    ([700, 650, 900, 910], (12, 2, 64), 64, [0, 2, 4], [640, 832], 300, 4, 0.0, True, {(0, 2), (2, 2)}),
    ([700, 650, 670], (8, 2, 128), 64, [0, 3], [640], 5000, 4, 0.0, False, {(0, 3)}),
    ([700, 650, 670], (8, 2, 128), 64, [0, 3], [640], 100, 300, 0.0, True, {(0, 3)}),
    ([3000, 2500, 2600, 2999], (6, 2, 128), 128, [1, 4], [2432], 0, 0, 20.0, False, {(1, 3)}),
    ([1500, 1510, 1520, 1530, 1540], (10, 1, 64), 32, [0, 5], [1472], 700, 0, 0.0, True, {(0, 3), (3, 2)}),
]


@pytest.mark.parametrize("c", FORMS, ids=lambda c: f"{len(c[0])}x{c[0][0]}-{c[1]}-p{c[2]}-{c[4]}-w{c[5]}-cap{c[7]}-bias{c[8]}")
def test_shared_forms(gpu, c):
    lengths, shape, page, starts, prefix, window, shared, cap, bias, want_tiles = c
    n = len(lengths)
    laid = pr.Laid(lengths, shape[1], shape[2], page, starts, prefix, seed=1)
    got, want, tol, plan = decode(gpu, laid, shape, lengths, list(range(n)), starts, prefix, window, shared, softcap=cap,
                                  bias=bias, row_none=True)
    assert set(tiles(plan, n)) == want_tiles
    covered(plan, n, shape[0] // shape[1])
    close(got, want, tol)


def test_pages_of_a_prefix_that_are_not_there(gpu):
    """A page that a group shares is missing: all its rows are NaN; one of a row's own: that row. A table row that is
    missing: the others of its group do without sharing."""
    shape, page = (8, 2, 128), 64
    lengths, starts, prefix = [800, 810, 700, 710, 705, 850, 70], [0, 2, 5], [768, 640]
    laid = pr.Laid(lengths, 2, 128, page, starts, prefix, seed=6)
    cache, q = laid.cache(), queries(5, 7, 8, 128)
    want, tol = pr.attend(laid, q, lengths, list(range(7)), 128 ** -0.5)

    def run(row, table):
        plan = gpu.page_plan(ints(lengths), ints(row), ints(table.tolist()), 8, cache, 850, starts=ints(starts),
                             prefix=ints(prefix))
        return plan, gpu.attn_decode_paged(q.cuda().view(-1), 0, 1024, cache, plan, 8, 128 ** -0.5).view(7, 8, 128)

    for bad in (-1, laid.pages, 2**31 - 1, -2**31):
        table = laid.table.clone()
        table[2:5, 7] = bad  # what a group shares
        table[5, 1] = bad    # a row's own
        plan, got = run([0, 1, 2, 3, 4, 5, bad if bad < 0 else 7], table)
        assert set(tiles(plan, 7)) == {(0, 2), (2, 3)}
        assert torch.isnan(got[2:]).all()
        close(got[:2], want[:2], tol[:2])
    plan, got = run([0, -5, 2, 3, 4, 5, 6], laid.table)
    assert set(tiles(plan, 7)) == {(2, 3)}
    assert torch.isnan(got[1]).all()
    at = [0, 2, 3, 4, 5, 6]
    close(got[at], want[at], tol[at])


@pytest.mark.parametrize("starts,prefix,some", [
    ([3, 1, 4], [704, 704], False), ([0, 4], [704 + 31], True), ([-5, 99], [704], True), ([0, 4], [-7], False),
    ([0, 4], [-2**31], False), ([4, 4], [704], False), ([-2**31, 2, 2**31 - 1], [704, 31], True),
    ([0, 2, 2, 4], [704, 704, 704], True), ([2, 3, 4], [704, 704], False)])
def test_groups_out_of_range(gpu, starts, prefix, some):
    """Starts that decrease, are empty or pass the rows; prefixes below 0 or that end within a block."""
    lengths = [730, 740, 750, 760]
    laid = pr.Laid(lengths, 2, 64, 32, [0, 4], [704], seed=7)
    got, want, tol, plan = decode(gpu, laid, (4, 2, 64), lengths, [0, 1, 2, 3], starts, prefix, bias=True)
    assert bool(tiles(plan, 4)) == some
    covered(plan, 4, 2)
    close(got, want, tol)


def test_prefix_past_the_shortest_row(gpu):
    """A prefix of more positions than there are counts up to the shortest row's length, in whole blocks."""
    lengths = [704, 720, 730]
    laid = pr.Laid([736] * 3, 2, 64, 32, [0, 3], [736], seed=7)
    got, want, tol, plan = decode(gpu, laid, (4, 2, 64), lengths, [0, 1, 2], [0, 3], [2**31 - 1], max_tk=736)
    assert tiles(plan, 3) and sorted(covered(plan, 3, 2)[0]) == list(range(22))
    close(got, want, tol)


def test_not_finite_within_groups(gpu):
    """Values that are not finite in what a group shares and in one row's own part; a NaN and an infinity in two
    rows' queries: their heads alone."""
    heads, kv, hd, page, n = 8, 2, 128, 32, 11
    lengths = [768 + 3 * t for t in range(n)]
    laid = pr.Laid(lengths, kv, hd, page, [0, n], [768], seed=3)
    laid.pool[1][torch.isnan(laid.pool[1])] = math.inf  # what no row sees
    q = queries(5, n, heads, hd)
    want, tol = pr.attend(laid, q, lengths, list(range(n)), 0.09)
    odd = q.clone()
    odd[5, 2, 7], odd[8, 6, 0] = math.nan, math.inf
    rest = torch.ones(n, heads, dtype=torch.bool)
    rest[5, 2] = rest[8, 6] = False

    def run(x):
        cache = laid.cache()
        plan = gpu.page_plan(ints(lengths), None, ints(laid.table.tolist()), heads, cache, 800, starts=ints([0, n]),
                             prefix=ints([768]))
        assert set(tiles(plan, n)) == {(0, 8), (8, 3)}
        return gpu.attn_decode_paged(x.cuda().view(-1), 0, heads * hd, cache, plan, heads, 0.09).view(n, heads, hd).cpu()

    got = run(odd)
    assert got[~rest].isnan().all()
    close(got[rest], want[rest], tol[rest])
    put(laid, 0, 100, 3, math.inf)
    put(laid, 0, 700, 4, math.nan)
    put(laid, 9, 790, 7, -math.inf)
    want, tol = pr.attend(laid, q, lengths, list(range(n)), 0.09)
    assert torch.isinf(want[:, 0, 3]).all() and torch.isinf(want[9, 0, 7]) and torch.isfinite(want[8, 0, 7])
    close(run(q), want, tol)


@pytest.mark.parametrize("far", [60.0, 400.0])
def test_not_finite_values_of_little_weight(gpu, far):
    """A value that is not finite and seen is in the context whatever its weight: its element is not finite, the
    others are the plain form's."""
    heads, kv, hd, page, n = 4, 1, 64, 32, 9
    lengths = [740 + t for t in range(n)]
    laid = pr.Laid(lengths, kv, hd, page, [0, n], [704], seed=3)
    laid.pool[1][torch.isnan(laid.pool[1])] = math.inf
    for j, dim in ((3, 5), (600, 6), (735, 7)):  # (the last in each row's own part)
        for t in range(n) if j > 704 else [0]:
            put(laid, t, j, dim, math.inf)
            x = int(laid.table[t, j // page])
            laid.pool[0, x, 0, j % page] = 0.0
            laid.pool[0, x, 0, j % page, 0] = -far
    for t in range(n):
        for j in (3, 600, 735):
            laid.k[t][0, j] = 0.0
            laid.k[t][0, j, 0] = -far
    q = queries(5, n, heads, hd)
    q[:, :, 0] = 4.0
    cache, table = laid.cache(), ints(laid.table.tolist())
    plan = gpu.page_plan(ints(lengths), None, table, heads, cache, 750, starts=ints([0, n]), prefix=ints([704]))
    assert set(tiles(plan, n)) == {(0, 8), (8, 1)}
    chosen = torch.arange(24, dtype=torch.int32).expand(n, kv, -1).contiguous().cuda()
    a = gpu.attn_decode_paged(q.cuda().view(-1), 0, heads * hd, cache, plan, heads, 1.0)
    b = gpu.attn_decode_selected(q.cuda().view(-1), 0, heads * hd, cache, table, None, ints(lengths), chosen, heads, 1.0)
    want, tol = pr.attend(laid, q, lengths, list(range(n)), 1.0)
    rest = torch.ones(hd, dtype=torch.bool)
    rest[5:8] = False
    for got in (a, b):
        got = got.view(n, heads, hd).cpu()
        assert not torch.isfinite(got[:, :, 5:8]).any()
        close(got[:, :, rest], want[:, :, rest], tol[:, :, rest])


def test_groups_from_a_graph(gpu):
    """A step whose groups, prefixes and lengths change between replays."""
    heads, kv, hd, page, cols, n = 8, 2, 128, 32, 32, 12
    laid = pr.Laid([cols * page] * n, kv, hd, page, [0, 5, n], [896, 768], seed=3)
    cache, table = laid.cache(), ints(laid.table.tolist())
    q = queries(5, n, heads, hd)
    dq, tk, starts, prefix = q.cuda().view(-1), ints([1] * n), ints([0, 5, n]), ints([0, 0])

    def step():
        plan = gpu.page_plan(tk, None, table, heads, cache, cols * page, starts=starts, prefix=prefix, window=900, shared=8)
        return plan.data, gpu.attn_decode_paged(dq, 0, heads * hd, cache, plan, heads, 0.09, 20.0, sl)

    sl = slopes_of(heads).cuda()
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        data, held = step()
    r = random.Random(3)
    for s, p in (([0, 5, n], [896, 768]), ([0, 4, 5], [896, 0]), ([5, n, n], [704, 0]), ([1, 5, n], [672, 32]), ([n, n, n], [0, 0])):
        lengths = [r.randint(p[0] if t < 5 else p[1], cols * page) for t in range(n)]
        for dev, host in ((tk, lengths), (starts, s), (prefix, p)):
            dev.copy_(torch.tensor(host, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        close(held, *pr.attend(laid, q, lengths, list(range(n)), 0.09, 20.0, slopes_of(heads), window=900, shared=8), what=(s, p))
        again, eager = step()
        assert torch.equal(held, eager) and torch.equal(data[:11], again[:11])  # (a plan's header is 11 words)


@pytest.mark.parametrize("seed", range(10))
def test_shared_random(gpu, seed):
    """Rows of sequences behind documents, in groups of any bounds, with the scores, windows and first positions of any
    kind: every block that a row needs is in one item of its own, and its context is the plain form's."""
    r = random.Random(100 + seed)
    kv, group, hd = r.choice([1, 2, 3]), r.choice([1, 2, 3, 4, 5, 6, 8, 10, 12, 16]), r.choice([64, 128])
    page, per = r.choice([32, 64, 128]), 32 // group
    cuts, prefix, lens = [0], [], []
    for _ in range(r.randint(1, 3)):
        doc = page * r.randint(-(-700 // page), 1200 // page)
        lens += [doc + r.choice([0, 1, 31, 32, 33, r.randint(0, 300)]) for _ in range(r.choice([1, 2, per, per + 1]))]
        cuts.append(len(lens))
        prefix.append(doc)
    laid = pr.Laid(lens, kv, hd, page, cuts, prefix, seed=seed)
    row, tk, starts = [], [], [0]
    for a, b in zip(cuts, cuts[1:]):
        for t in range(a, b):
            m = r.choice([1, 1, 1, 2, 3, per])
            row += [t] * m
            tk += [max(0, lens[t] - m + 1 + j) for j in range(m)]
        starts.append(len(row))
    window, shared = r.choice([0, 0, 0, r.randint(1, 1200)]), r.choice([0, 5, 100])
    lo = [r.randint(0, 600) for _ in row] if r.random() < 0.3 else None
    got, want, tol, plan = decode(gpu, laid, (kv * group, kv, hd), tk, row, starts, prefix, window, shared, lo,
                                  r.choice([0.0, 20.0]), r.random() < 0.6, seed=seed)
    for t, blocks in enumerate(covered(plan, len(row), group)):
        need = {int(j) // 32 for j in pr.seen_of(tk[t], lo[t] if lo else 0, window, shared, tk[t]).nonzero()}
        assert len(set(blocks)) == len(blocks) and need <= set(blocks), t
    close(got, want, tol)
