"""The paged cache's operators: attention over pages with shared prefixes and
over selected pages, the pages' key bounds and their selection, the store,
against plain 64-bit forms."""
import math
import random

import pytest
import torch

import paged_ref as pr
import ranges_ref as ref
from test_ranges_gpu import close, slopes_of

pytestmark = pytest.mark.gpu


def ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32).cuda()


def queries(seed, rows, heads, hd, scale=2.0):
    return scale * torch.randn(rows, heads, hd, generator=torch.Generator().manual_seed(seed))


def decode(gpu, laid, shape, tk, row, starts=None, prefix=None, window=0, shared=0, lo=None, softcap=0.0, bias=False,
           max_tk=None, seed=5, table=None, row_none=False):
    heads, kv, hd = shape
    q = queries(seed, len(tk), heads, hd)
    sl = slopes_of(heads) if bias else None
    cache = laid.cache()
    plan = gpu.page_plan(ints(tk), None if row_none else ints(row), ints((laid.table if table is None else table).tolist()),
                         heads, cache, max_tk or max(max(tk), 1), starts=ints(starts), prefix=ints(prefix),
                         lo_dev=ints(lo), window=window, shared=shared)
    got = gpu.attn_decode_paged(q.cuda().view(-1), 0, heads * hd, cache, plan, heads, hd ** -0.5, softcap,
                                None if sl is None else sl.cuda())
    want, tol = pr.attend(laid, q, tk, row, hd ** -0.5, softcap, sl, lo, window, shared)
    return got, want, tol, plan


# lengths, (heads, kv, hd), page, groups' first rows, prefixes, window, shared, softcap, bias
DECODE = [
    ([1], (4, 4, 64), 32, None, None, 0, 0, 0.0, False),
    ([0, 5, 33], (8, 2, 128), 32, None, None, 0, 0, 50.0, True),
    ([700], (8, 2, 128), 64, None, None, 0, 0, 0.0, False),
    ([2300, 40], (4, 1, 64), 128, None, None, 0, 0, 0.0, True),
    ([9000], (8, 8, 128), 256, None, None, 0, 0, 30.0, False),
    ([130, 129, 128], (8, 2, 128), 64, [0, 3], [128], 0, 0, 0.0, False),
    ([130, 200], (32, 8, 128), 32, [0, 2], [128], 0, 0, 0.0, True),
    ([400, 500, 385, 384, 600, 390, 391, 392, 393], (8, 2, 128), 128, [0, 9], [384], 0, 0, 50.0, True),
    ([300] * 33 + [17], (4, 4, 64), 32, [0, 33], [256], 0, 0, 0.0, False),
    ([700, 650, 130, 64, 64, 900, 910], (16, 1, 128), 64, [0, 2, 3, 5, 7], [640, 128, 64, 832], 0, 0, 30.0, False),
    ([700, 650, 900, 910], (12, 2, 64), 64, [0, 2, 4], [640, 832], 300, 4, 0.0, True),
    ([700, 650, 670], (8, 2, 128), 64, [0, 3], [640], 5000, 4, 0.0, False),
    ([700, 650, 670], (8, 2, 128), 64, [0, 3], [640], 100, 300, 0.0, False),
    ([700, 650, 670], (8, 2, 128), 32, [0, 3], [640], 20, 0, 0.0, False),
    ([3000, 2500, 2600, 2999], (6, 2, 128), 128, [1, 4], [2432], 0, 0, 0.0, False),
]


@pytest.mark.parametrize("c", DECODE, ids=lambda c: f"{len(c[0])}x{c[0][0]}-{c[1]}-p{c[2]}-{c[4]}-w{c[5]}-cap{c[7]}-bias{c[8]}")
def test_decode(gpu, c):
    lengths, shape, page, starts, prefix, window, shared, cap, bias = c
    laid = pr.Laid(lengths, shape[1], shape[2], page, starts, prefix, seed=1)
    got, want, tol, _ = decode(gpu, laid, shape, lengths, list(range(len(lengths))), starts, prefix, window, shared,
                               softcap=cap, bias=bias, row_none=True)
    close(got, want, tol)
    for r, n in enumerate(lengths):
        if n == 0:
            assert not got.view(want.shape)[r].any()


def covered(plan, nseq, group):
    """For each row the blocks that its items walk, in the plan's words."""
    d = plan.data.cpu().tolist()
    total, wide = d[0], d[1]
    at = (16 + 12 * nseq + 15) // 16 * 16
    items = [d[at + 16 * i:at + 16 * i + 16] for i in range(total)]
    got = [[] for _ in range(nseq)]
    for i, e in enumerate(items):
        na, b0, c0, d0 = e[4:8]
        blocks = [b if b < na else b0 + b - na if b - na < c0 - b0 else d0 + b - na - (c0 - b0) for b in range(e[8], e[9])]
        for r in range(e[0], e[0] + e[1]):
            got[r] += blocks
        assert e[1] * group <= 32 and (i < wide or e[1] == 1)
    for r in range(nseq):
        o0, on, s0, sn, step, col, own = d[16 + 12 * r:16 + 12 * r + 7]
        for j in range(on):
            e = items[o0 + j if own >= 0 else wide + o0 + j]
            assert e[0] + max(own, 0) // group == r and e[3] & 2 == 0 and (own < 0 or o0 + j < wide)
        for j in range(sn):
            e = items[s0 + j * step]
            assert s0 + j * step < wide and e[3] & 2 and e[0] + col // group == r and col % group == 0
    return got


@pytest.mark.parametrize("seed", range(10))
def test_decode_random(gpu, seed):
    r = random.Random(seed)
    n, page = r.randint(1, 24), r.choice([32, 64, 128])
    shape = r.choice([(8, 2, 128), (4, 4, 64), (12, 4, 64), (5, 5, 128), (16, 1, 128)])
    cuts = sorted(r.choices(range(n + 1), k=r.randint(2, 5)))
    prefix = [page * r.randint(0, 800 // page) for _ in cuts[1:]]
    lengths = [r.randint(0, 600) for _ in range(n)]
    for a, b, p in zip(cuts, cuts[1:], prefix):
        for t in range(a, b):
            lengths[t] += p
    window, shared = r.choice([0, 0, r.randint(1, 900)]), r.choice([0, 5, 100])
    lo = [r.randint(0, max(lengths[0], 1)) for _ in lengths] if r.random() < 0.3 else None
    laid = pr.Laid(lengths, shape[1], shape[2], page, cuts, prefix, seed=seed)
    got, want, tol, plan = decode(gpu, laid, shape, lengths, list(range(n)), cuts, prefix, window, shared, lo,
                                  r.choice([0.0, 20.0]), r.random() < 0.4)
    close(got, want, tol, (lengths, cuts, prefix, window, shared, shape, page))
    for t, blocks in enumerate(covered(plan, n, shape[0] // shape[1])):
        m = lengths[t]
        seen = pr.seen_of(m, lo[t] if lo else 0, window, shared, m)
        need = sorted({int(j) // 32 for j in seen.nonzero()})
        assert sorted(set(blocks)) == sorted(blocks), "a block twice"
        assert set(need) <= set(blocks), (t, need, blocks)


def test_rows_of_prompts(gpu):
    """Rows of two sequences behind one document, each row one position further."""
    shape, page, per = (8, 2, 128), 64, 21
    laid = pr.Laid([512 + per, 512 + per + 9], 2, 128, page, [0, 2], [512], seed=3)
    tk = [512 + j + 1 for j in range(per)] + [512 + 9 + j + 1 for j in range(per)]
    row = [0] * per + [1] * per
    got, want, tol, _ = decode(gpu, laid, shape, tk, row, [0, 2 * per], [512])
    close(got, want, tol)


def test_many_rows_and_groups(gpu):
    """Groups past one wave of the plan's threads, rows past its workgroup."""
    n = 1500
    lengths = [64 + (7 * i) % 40 for i in range(n)]
    starts = list(range(0, n + 1, 2))
    laid = pr.Laid(lengths, 1, 64, 32, starts, [64] * 750, seed=4)
    got, want, tol, plan = decode(gpu, laid, (2, 1, 64), lengths, list(range(n)), starts, [64] * 750)
    close(got, want, tol)
    covered(plan, n, 2)


def test_bad_rows_and_pages(gpu):
    """A table row that is not there, a page that is not there: NaN, and nobody else's context."""
    shape, page = (8, 2, 128), 64
    lengths = [300, 310, 200, 210, 205, 150, 70]
    starts, prefix = [0, 2, 5], [256, 128]
    laid = pr.Laid(lengths, 2, 128, page, starts, prefix, seed=6)
    for bad in (-1, laid.pages, 2**31 - 1, -2**31):
        table = laid.table.clone()
        table[5, 1] = bad       # a row's own
        table[2:5, 0] = bad     # what a group shares
        row = [0, 1, 2, 3, 4, 5, 6]
        q = queries(5, 7, 8, 128)
        cache = laid.cache()
        plan = gpu.page_plan(ints(lengths), ints(row[:6] + [bad if bad < 0 else 7]), ints(table.tolist()), 8, cache, 310,
                             starts=ints(starts), prefix=ints(prefix))
        got = gpu.attn_decode_paged(q.cuda().view(-1), 0, 1024, cache, plan, 8, 128 ** -0.5).view(7, 8, 128)
        want, tol = pr.attend(laid, q, lengths, row, 128 ** -0.5)
        assert torch.isnan(got[2:]).all()
        close(got[:2], want[:2], tol[:2])
    # A bad row in a group: its others do without sharing.
    q = queries(5, 7, 8, 128)
    plan = gpu.page_plan(ints(lengths), ints([0, -5, 2, 3, 4, 5, 6]), ints(laid.table.tolist()), 8, cache, 310,
                         starts=ints(starts), prefix=ints(prefix))
    got = gpu.attn_decode_paged(q.cuda().view(-1), 0, 1024, cache, plan, 8, 128 ** -0.5).view(7, 8, 128)
    assert torch.isnan(got[1]).all()
    at = [0, 2, 3, 4, 5, 6]
    close(got[at], want[at], tol[at])


def test_plan_of_odd_groups(gpu):
    """Starts that decrease or pass the rows, prefixes past the rows and below 0, lengths past the table."""
    shape, lengths = (4, 2, 64), [200, 210, 220, 230]
    laid = pr.Laid(lengths, 2, 64, 32, [0, 4], [192], seed=7)
    for starts, prefix in (([3, 1, 4], [192, 192]), ([0, 4], [10**9]), ([-5, 99], [192]), ([0, 4], [-7]), ([4, 4], [192])):
        cap = prefix if prefix != [10**9] else [192]
        if prefix == [10**9]:  # their tables agree no further
            laid2 = pr.Laid([192 + i for i in range(4)], 2, 64, 32, [0, 4], [192], seed=7)
            got, want, tol, _ = decode(gpu, laid2, shape, [192] * 4, [0, 1, 2, 3], starts, prefix)
        else:
            got, want, tol, _ = decode(gpu, laid, shape, lengths, [0, 1, 2, 3], starts, cap)
        close(got, want, tol, (starts, prefix))
    got, want, tol, _ = decode(gpu, pr.Laid([64, 64], 2, 64, 32, seed=1), shape, [64, 64], [0, 1], max_tk=64)
    q = queries(5, 2, 4, 64)
    laid = pr.Laid([64, 64], 2, 64, 32, seed=1)
    cache = laid.cache()
    plan = gpu.page_plan(ints([10**9, -3]), None, ints(laid.table.tolist()), 4, cache, 64)
    got = gpu.attn_decode_paged(q.cuda().view(-1), 0, 256, cache, plan, 4, 0.125).view(2, 4, 64)
    close(got[0], want[0], tol[0])
    assert not got[1].any()


def test_plan_of_other_sizes(gpu):
    """A plan that another batch was made with gives NaN, not a context."""
    laid = pr.Laid([100, 200], 2, 64, 32, seed=1)
    cache = laid.cache()
    plan = gpu.page_plan(ints([100, 200]), None, ints(laid.table.tolist()), 4, cache, 200)
    other = gpu.page_plan(ints([100]), None, ints(laid.table[:1].tolist()), 4, cache, 200)
    plan.data = torch.cat([other.data, other.data.new_zeros(plan.data.numel() - other.data.numel())])
    q = queries(1, 2, 4, 64)
    assert torch.isnan(gpu.attn_decode_paged(q.cuda().view(-1), 0, 256, cache, plan, 4, 0.125)).all()


def test_not_finite_values(gpu):
    """Infinities of keys and values that a row sees are in its context; those of others are not."""
    lengths = [130, 140]
    laid = pr.Laid(lengths, 2, 64, 32, [0, 2], [128], seed=8)
    laid.pool[1][torch.isnan(laid.pool[1])] = math.inf
    t = int(laid.table[1, 4])
    laid.pool[1, t, 0, 3, 5] = math.inf  # position 131 of the second row
    laid.v[1][0, 131, 5] = math.inf
    got, want, tol, _ = decode(gpu, laid, (4, 2, 64), lengths, [0, 1], [0, 2], [128])
    close(got, want, tol)
    assert torch.isinf(want[1, :2, 5]).all()


def test_far_pages(gpu):
    """Pages whose bytes lie past 2^32 in the cache."""
    kv, hd, page = 8, 128, 4096
    pages = 70  # 2^26 bytes each
    from ttsxabe_amd.gpu import PagedCache16
    cache = PagedCache16(kv, hd, pages, page, zero=False)
    laid = pr.Laid([5000], kv, hd, page, seed=9, spare=0)
    small = ref.tile(laid.pool[0], laid.pool[1]).view(2, -1)
    cache.data.view(pages, -1)[68:70] = small.cuda()
    table = laid.table + 68
    q = queries(2, 1, kv, hd)
    plan = gpu.page_plan(ints([5000]), None, ints(table.tolist()), kv, cache, 5000)
    got = gpu.attn_decode_paged(q.cuda().view(-1), 0, kv * hd, cache, plan, kv, hd ** -0.5)
    want, tol = pr.attend(laid, q, [5000], [0], hd ** -0.5)
    close(got, want, tol)
    bounds = torch.zeros(pages, kv, 2, hd, dtype=torch.float16).cuda()
    gpu.page_bounds(cache, ints(table.tolist()), None, None, ints([5000]), 5000, bounds)
    for p in range(2):
        assert torch.equal(bounds[int(table[0, p])].float().cpu(), pr.bounds(laid, 0, 5000, p))


# ------------------------------------------------------------ selected pages

SELECTED = [
    # lengths, rows of each, shape, page, pages of each row, softcap, bias
    ([1], 1, (4, 4, 64), 32, 1, 0.0, False),
    ([700, 90], 1, (8, 2, 128), 64, 4, 0.0, True),
    ([5000], 1, (8, 2, 128), 64, 20, 50.0, False),
    ([900, 1300], 9, (16, 1, 64), 32, 7, 0.0, False),
    ([2000], 3, (5, 5, 128), 256, 3, 0.0, True),
    ([300], 70, (32, 8, 128), 32, 5, 30.0, False),
]


@pytest.mark.parametrize("c", SELECTED, ids=lambda c: f"{len(c[0])}x{c[1]}x{c[0][0]}-{c[2]}-p{c[3]}-{c[4]}")
def test_selected(gpu, c):
    lengths, per, shape, page, count, cap, bias = c
    heads, kv, hd = shape
    laid = pr.Laid(lengths, kv, hd, page, seed=1)
    tk = [max(1, n - per + 1 + j) for n in lengths for j in range(per)]
    row = [t for t in range(len(lengths)) for _ in range(per)]
    r = random.Random(2)
    chosen = torch.full((len(tk), kv, count), -1, dtype=torch.int32)
    for i, m in enumerate(tk):
        for h in range(kv):
            live = (m + page - 1) // page
            ids = r.sample(range(live + 2), min(count, live))  # in no order, some past the row's positions
            chosen[i, h, :len(ids)] = torch.tensor(ids)
    chosen[0, 0] = torch.tensor([-1, -5, 10**9][:count] + [-1] * (count - 3))  # nothing
    q = queries(3, len(tk), heads, hd)
    sl = slopes_of(heads) if bias else None
    got = gpu.attn_decode_selected(q.cuda().view(-1), 0, heads * hd, laid.cache(), ints(laid.table.tolist()), ints(row),
                                   ints(tk), chosen.cuda(), heads, hd ** -0.5, cap, None if sl is None else sl.cuda())
    want, tol = pr.attend(laid, q, tk, row, hd ** -0.5, cap, sl, chosen=chosen)
    close(got, want, tol)
    assert not got.view(want.shape)[0, :heads // kv].any()


@pytest.mark.parametrize("lengths,count", [([300, 200, 100], 4), ([2000], 40)])
def test_selected_bad(gpu, lengths, count):
    laid = pr.Laid(lengths + [90], 2, 64, 32, seed=1)
    table = laid.table.clone()
    table[0, 1] = laid.pages  # needed by row 0 alone
    n = len(lengths) + 1
    chosen = torch.arange(count, dtype=torch.int32).expand(n, 2, -1).contiguous()
    q = queries(3, n, 4, 64)
    row = list(range(n - 1)) + [-1]
    got = gpu.attn_decode_selected(q.cuda().view(-1), 0, 256, laid.cache(), ints(table.tolist()), ints(row),
                                   ints(lengths + [90]), chosen.cuda(), 4, 0.125).view(n, 4, 64)
    want, tol = pr.attend(laid, q, lengths + [90], list(range(n)), 0.125, chosen=chosen)
    assert torch.isnan(got[0]).all() and torch.isnan(got[-1]).all()
    close(got[1:-1], want[1:-1], tol[1:-1])


def test_selected_all_is_decode(gpu):
    """All pages selected: what attention over all positions gives."""
    shape, lengths = (8, 2, 128), [1000, 777]
    laid = pr.Laid(lengths, 2, 128, 64, seed=2)
    got, want, tol, _ = decode(gpu, laid, shape, lengths, [0, 1])
    chosen = torch.arange(16, dtype=torch.int32).expand(2, 2, -1).contiguous().cuda()
    q = queries(5, 2, 8, 128)
    sel = gpu.attn_decode_selected(q.cuda().view(-1), 0, 1024, laid.cache(), ints(laid.table.tolist()), None, ints(lengths),
                                   chosen, 8, 128 ** -0.5)
    close(sel, want, tol)


# ------------------------------------------------------------------- bounds

@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("page", [32, 64, 256])
@pytest.mark.parametrize("kv", [1, 5])
def test_bounds(gpu, hd, page, kv):
    lengths = [1, page, page + 1, 0, 5 * page - 7, 700]
    laid = pr.Laid(lengths, kv, hd, page, seed=3)
    cache, table = laid.cache(), ints(laid.table.tolist())
    low = [0, page - 1, 0, 0, 2 * page, 699]
    start = torch.full((laid.pages, kv, 2, hd), 7.0, dtype=torch.float16).cuda()
    for new in (1, 10000):  # more positions than were said: taken all the same
        got = start.clone()
        gpu.page_bounds(cache, table, None, ints(low), ints(lengths), new, got)
        want = start.clone().float().cpu()
        for t, (a, b) in enumerate(zip(low, lengths)):
            for p in range(a // page, (b + page - 1) // page if a < b else 0):
                want[int(laid.table[t, p])] = pr.bounds(laid, t, b, p)
        assert torch.equal(got.float().cpu(), want)
    # Rows and pages that are not there are passed over.
    bad = laid.table.clone()
    bad[4, 3] = laid.pages
    got = start.clone()
    gpu.page_bounds(cache, ints(bad.tolist()), ints([-1, 6, 4]), None, ints([10, 10, lengths[4]]), 1, got)
    want = start.clone().float().cpu()
    for p in (0, 1, 2, 4):
        want[int(laid.table[4, p])] = pr.bounds(laid, 4, lengths[4], p)
    assert torch.equal(got.float().cpu(), want)


def test_bounds_not_finite(gpu):
    laid = pr.Laid([40], 2, 64, 32, seed=3)
    x = int(laid.table[0, 0])
    laid.pool[0, x, 0, 5, 7], laid.pool[0, x, 1, 31, 63], laid.pool[0, x, 1, 2, 9] = math.nan, math.inf, -math.inf
    got = torch.zeros(laid.pages, 2, 2, 64, dtype=torch.float16).cuda()
    gpu.page_bounds(laid.cache(), ints(laid.table.tolist()), None, None, ints([40]), 40, got)
    b = got[x].cpu().float()
    assert b[0, :, 7].isnan().all() and not b[0, :, :7].isnan().any() and b[1, 0, 63] == math.inf and b[1, 1, 9] == -math.inf


# ---------------------------------------------------------------- selection

SELECT = [
    # pages of the sequences, rows of each, shape, page, count, first, last
    ([3], 1, (4, 4, 64), 32, 5, 1, 1),
    ([40, 7, 100], 1, (8, 2, 128), 64, 9, 1, 2),
    ([300], 2, (16, 1, 64), 32, 1, 0, 1),
    ([2500], 1, (4, 2, 128), 32, 60, 0, 0),
    ([70], 13, (12, 4, 128), 128, 32, 2, 3),
    ([33, 34], 1, (5, 5, 64), 256, 33, 33, 0),
]


@pytest.mark.parametrize("c", SELECT, ids=lambda c: f"{c[0]}x{c[1]}-{c[2]}-{c[4]}")
def test_select(gpu, c):
    wide, per, (heads, kv, hd), page, count, first, last = c
    g = torch.Generator().manual_seed(4)
    pages, cols = sum(wide) + 2, max(wide)
    mid, half = torch.randn(pages, kv, 1, hd, generator=g), 1.0 + torch.randn(pages, kv, 1, hd, generator=g).abs()
    bounds = torch.cat([mid + half, mid - half], 2).to(torch.float16)
    order = torch.randperm(pages, generator=g)
    table, at = [], 0
    for w in wide:
        table.append(order[at:at + w].tolist() + [-1] * (cols - w))
        at += w
    table = torch.tensor(table)
    tk = [max(0, w * page - 3 - 5 * j) for w in wide for j in range(per)]
    row = [t for t in range(len(wide)) for _ in range(per)]
    q = queries(6, len(tk), heads, hd)
    want = pr.select(q, bounds, table, row, tk, page, count, first, last)
    got = gpu.select_pages(q.cuda().view(-1), 0, heads * hd, bounds.cuda(), ints(table.tolist()), ints(row), ints(tk),
                           cols * page, heads, page, count, first, last)
    assert torch.equal(got.cpu(), want)


def test_select_ties_and_not_finite(gpu):
    """Equal pages: the lowest; NaN and missing pages first; rows that are not there: none."""
    heads, kv, hd, page, n = 4, 2, 64, 32, 50
    g = torch.Generator().manual_seed(1)
    one = torch.randn(1, kv, 2, hd, generator=g).to(torch.float16)
    bounds = one.expand(n, -1, -1, -1).clone()
    q = queries(6, 3, heads, hd)
    table = torch.arange(n).expand(2, -1).clone()
    tk, row = [n * page, n * page - 31, 10], [0, 1, 2]

    def run(b, t):
        want = pr.select(q, b, t, row, tk, page, 6, 1, 1)
        got = gpu.select_pages(q.cuda().view(-1), 0, heads * hd, b.cuda(), ints(t.tolist()), ints(row), ints(tk), n * page,
                               heads, page, 6, 1, 1)
        assert torch.equal(got.cpu(), want)
        return want

    want = run(bounds, table)
    assert want[0, 0].tolist() == [0, 1, 2, 3, 4, 49] and want[2].max() == -1
    bounds[17, :, 0, 3] = math.nan
    bounds[21] = math.inf
    table[1, 30] = n
    want = run(bounds, table)
    assert 17 in want[0, 0].tolist() and 30 in want[1, 1].tolist()
    bounds[:] = 0.0  # and a zero query: all scores 0 or -0
    bounds[::2, :, 0] = -0.0
    run(bounds, table)
    big = one.expand(n, -1, -1, -1).clone()
    big[:, :, 0], big[:, :, 1] = 65504.0, -65504.0
    q = 1e30 * queries(6, 3, heads, hd)
    run(big, table)


def test_select_clamps_to_max_tk(gpu):
    """Lengths past max_tk count as it."""
    heads, kv, hd, page, n = 2, 1, 64, 32, 40
    g = torch.Generator().manual_seed(1)
    bounds = torch.randn(n, kv, 2, hd, generator=g).to(torch.float16)
    q = queries(6, 1, heads, hd)
    table = torch.arange(n)[None]
    got = gpu.select_pages(q.cuda().view(-1), 0, heads * hd, bounds.cuda(), ints(table.tolist()), None, ints([10**9]),
                           20 * page, heads, page, 6, 1, 1)
    assert torch.equal(got.cpu(), pr.select(q, bounds, table, [0], [20 * page], page, 6, 1, 1))


# -------------------------------------------------------------------- store

@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("c", [
    (1, (4, 4, 64), 32, 64), (5, (8, 2, 128), 64, 96), (70, (4, 2, 64), 32, 64), (200, (8, 2, 128), 256, 128),
    (333, (4, 4, 128), 64, 64)], ids=str)
def test_store(gpu, c, inter):
    """Rows of three sequences, some padding: the same bits as the store into slots, pages taken as such."""
    from ttsxabe_amd.gpu import PagedCache16, TiledCache16
    rows, (heads, kv, hd), page, rot = c
    g = torch.Generator().manual_seed(1)
    cols, pages = (rows + 40 + page) // page + 1, 3 * ((rows + 40 + page) // page + 1)
    table = torch.randperm(pages, generator=g).view(3, cols).to(torch.int32)
    seq = torch.tensor([3 * r // rows for r in range(rows)], dtype=torch.int32)
    index = torch.arange(rows, dtype=torch.int32) + 13
    if rows > 4:
        seq[1], index[2], table[2, 0] = 3, cols * page, pages  # no such sequence, position, page
        seq[3], index[4] = -1, -1
    x = torch.randn(rows, (heads + 2 * kv) * hd, generator=g).cuda()
    n = pages * kv * page * 2 * hd
    start = torch.randn(n, generator=g).to(torch.float16).cuda()
    paged = PagedCache16.of(start.clone(), kv, hd, pages, page)
    slots = TiledCache16.of(start.clone(), kv, hd, page, slots=pages)
    q1, q2 = torch.empty(rows * heads * hd, device="cuda"), torch.empty(rows * heads * hd, device="cuda")
    width, pos = (heads + 2 * kv) * hd, index.cuda()
    div = torch.linspace(1.0, 3.0, rot // 2).cuda()
    gpu.paged_rope_store(x, 0, x, heads * hd, x, (heads + kv) * hd, width, pos, seq.cuda(), pos, table.cuda(), div, rows,
                         heads, rot, 1e4, 1.1, inter, paged, q_out=q1)
    good = (seq >= 0) & (seq < 3) & (index >= 0) & (index < cols * page)
    at = torch.where(good, index // page, 0).long()
    slot = torch.where(good, table[seq.clamp(0, 2).long(), at], -1).to(torch.int32)
    gpu.t16_rope_store(x, 0, x, heads * hd, x, (heads + kv) * hd, width, pos, slot.cuda(), (index % page).cuda(), div, rows,
                       heads, rot, 1e4, 1.1, inter, slots, q_out=q2)
    assert torch.equal(q1, q2) and torch.equal(paged.data.view(torch.int16), slots.data.view(torch.int16))
    assert not torch.equal(paged.data, start)
    k, v = ref.untile(paged.data.cpu(), pages, kv, hd, page)
    want = ref.rotate(x.cpu().view(rows, -1, hd)[:, heads:heads + kv], index.long(), rot, 1e4, div.cpu(), 1.1, inter)
    for r in range(rows):
        s = int(slot[r])
        if 0 <= s < pages:
            got = k[s, :, int(index[r]) % page].double()
            assert ((got - want[r]).abs() <= 2.0 ** -11 * want[r].abs() + 2.0 ** -19 * 8).all()
            assert torch.equal(v[s, :, int(index[r]) % page], x.cpu().view(rows, -1, hd)[r, heads + kv:].to(torch.float16))


# ------------------------------------------------------------------ together

def test_step_together(gpu):
    """Prompts stored page by page behind a shared document, then a step: the store, the bounds, the selection and
    both attentions, replayed from a graph as lengths grow."""
    from ttsxabe_amd.gpu import PagedCache16
    heads, kv, hd, page, doc, n = 8, 2, 128, 32, 256, 3
    cols = 20
    g = torch.Generator().manual_seed(2)
    cache = PagedCache16(kv, hd, 64, page)
    order = torch.randperm(64, generator=g).tolist()
    lead, rest = order[:doc // page], order[doc // page:]
    table = torch.tensor([lead + rest[12 * t:12 * t + 12] for t in range(n)], dtype=torch.int32)
    dt = table.cuda()
    keys = [torch.zeros(0, heads + 2 * kv, hd) for _ in range(n)]
    width = (heads + 2 * kv) * hd

    def store(x, seq, at):
        q = torch.empty(len(x) * heads * hd, device="cuda")
        i = ints(at)
        gpu.paged_rope_store(x, 0, x, heads * hd, x, (heads + kv) * hd, width, i, ints(seq), i, dt, None, len(x), heads,
                             hd, 1e4, 1.0, False, cache, q_out=q)
        return q

    document = torch.randn(doc, width, generator=g)
    store(document.cuda(), [0] * doc, list(range(doc)))
    first = [5, 40, 33]
    own = [torch.randn(m + 8, width, generator=g) for m in first]
    for t, m in enumerate(first):
        store(own[t][:m].cuda(), [t] * m, list(range(doc, doc + m)))
    bounds = torch.zeros(64, kv, 2, hd, dtype=torch.float16).cuda()
    gpu.page_bounds(cache, dt, None, None, ints([doc + m for m in first]), 300, bounds)

    x = torch.empty(n, width, device="cuda")
    at, tk = ints([0] * n), ints([0] * n)
    seq = ints(range(n))
    starts, prefix = ints([0, n]), ints([doc])
    q = torch.empty(n * heads * hd, device="cuda")
    low = torch.empty_like(at)

    def step():
        gpu.paged_rope_store(x, 0, x, heads * hd, x, (heads + kv) * hd, width, at, seq, at, dt, None, n, heads, hd, 1e4,
                             1.0, False, cache, q_out=q)
        gpu.page_bounds(cache, dt, None, at, tk, 1, bounds)
        plan = gpu.page_plan(tk, None, dt, heads, cache, cols * page, starts=starts, prefix=prefix)
        full = gpu.attn_decode_paged(q, 0, heads * hd, cache, plan, heads, hd ** -0.5)
        chosen = gpu.select_pages(q, 0, heads * hd, bounds, dt, None, tk, cols * page, heads, page, 5, 1, 2)
        some = gpu.attn_decode_selected(q, 0, heads * hd, cache, dt, None, tk, chosen, heads, hd ** -0.5)
        return full, chosen, some

    def check(got, i):
        full, chosen, some = got
        torch.cuda.synchronize()
        ks, vs = ref.untile(cache.data.cpu(), 64, kv, hd, page)
        laid = pr.Laid.__new__(pr.Laid)
        laid.page, laid.kv, laid.hd = page, kv, hd
        laid.k = [ks[table[t].long()].transpose(0, 1).reshape(kv, -1, hd) for t in range(n)]
        laid.v = [vs[table[t].long()].transpose(0, 1).reshape(kv, -1, hd) for t in range(n)]
        lens = [doc + m + i + 1 for m in first]
        for t, m in enumerate(first):  # what the step stored
            assert torch.equal(laid.v[t][:, lens[t] - 1].float(), own[t][m + i].view(-1, hd)[heads + kv:].to(torch.float16).float())
        qc = q.cpu().view(n, heads, hd)
        close(full, *pr.attend(laid, qc, lens, list(range(n)), hd ** -0.5))
        b = torch.zeros(64, kv, 2, hd)
        for t in range(n):
            for p in range((lens[t] + page - 1) // page):
                b[int(table[t, p])] = pr.bounds(laid, t, lens[t], p)
                assert torch.equal(bounds[int(table[t, p])].float().cpu(), b[int(table[t, p])])
        want = pr.select(qc, b, table, list(range(n)), lens, page, 5, 1, 2)
        assert torch.equal(chosen.cpu(), want)
        close(some, *pr.attend(laid, qc, lens, list(range(n)), hd ** -0.5, chosen=want))

    def load(i):
        x.copy_(torch.stack([own[t][m + i] for t, m in enumerate(first)]))
        at.copy_(torch.tensor([doc + m + i for m in first]))
        tk.copy_(at + 1)

    load(0)
    check(step(), 0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(1, 7):
        load(i)
        graph.replay()
        check(held, i)
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))


def test_streams(gpu):
    """Two calls at once on streams of their own."""
    shape, lengths = (8, 2, 128), [2000 + 100 * i for i in range(6)]
    laid = pr.Laid(lengths, 2, 128, 64, [0, 6], [1984], seed=1)
    cache, table = laid.cache(), ints(laid.table.tolist())
    q = [queries(i, 6, 8, 128).cuda().view(-1) for i in range(4)]
    tk, starts, prefix = ints(lengths), ints([0, 6]), ints([1984])
    torch.cuda.synchronize()
    plan = gpu.page_plan(tk, None, table, 8, cache, 2500, starts=starts, prefix=prefix)
    want = [gpu.attn_decode_paged(x, 0, 1024, cache, plan, 8, 0.09) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in q]
    got = [None] * 4
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = gpu.attn_decode_paged(q[i], 0, 1024, cache, plan, 8, 0.09)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("n,units", [(100, 1), (300, 1), (700, 40), (9000, 1)])
@pytest.mark.parametrize("hd", [64, 128])
def test_select_near_scores(gpu, n, units, hd):
    """Pages a step of f16 apart in a dim or two: few near the border, many, more than are held, by one workgroup
    and by several."""
    heads, kv, page = 4, 2, 32
    g = torch.Generator().manual_seed(n)
    one = torch.randn(1, kv, 1, hd, generator=g)
    bounds = torch.cat([one + 1.0, one - 1.0], 2).to(torch.float16).expand(n, -1, -1, -1).clone()
    at = torch.randint(0, hd, (n, 2), generator=g)
    bits = bounds.view(torch.int16)
    p = torch.arange(n)
    bits[p, 0, 0, at[:, 0]] += 1
    bits[p, 1, 1, at[:, 1]] -= 1
    if n == 700:  # and most of them far
        bounds[: n // 2] *= 0.5
    table = torch.randperm(n, generator=g)[None].expand(units, -1)
    tk = [n * page - r for r in range(units)]
    q = queries(7, units, heads, hd)
    want = pr.select(q[:2], bounds, table[:2], list(range(units))[:2], tk, page, 20, 1, 1)
    got = gpu.select_pages(q.cuda().view(-1), 0, heads * hd, bounds.cuda(), ints(table.tolist()), None, ints(tk),
                           n * page, heads, page, 20, 1, 1)
    assert torch.equal(got[:2].cpu(), want)


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e30])
def test_select_small_and_large_queries(gpu, scale):
    heads, kv, hd, page, n = 6, 2, 128, 64, 200
    g = torch.Generator().manual_seed(3)
    mid, half = torch.randn(n, kv, 1, hd, generator=g), torch.randn(n, kv, 1, hd, generator=g).abs()
    bounds = torch.cat([mid + half, mid - half], 2).to(torch.float16)
    bounds[5] *= 1000.0
    table = torch.arange(n)[None]
    q = queries(7, 1, heads, hd) * scale
    q[0, 1] *= 1e-6
    want = pr.select(q, bounds, table, [0], [n * page], page, 30, 0, 1)
    got = gpu.select_pages(q.cuda().view(-1), 0, heads * hd, bounds.cuda(), ints(table.tolist()), None, ints([n * page]),
                           n * page, heads, page, 30, 0, 1)
    assert torch.equal(got.cpu(), want)


def put(laid, t, j, dim, x):
    """x into dim `dim` of the value of kv head 0 at position j of sequence t, in its page (which others may share)."""
    p = int(laid.table[t, j // laid.page])
    laid.pool[1, p, 0, j % laid.page, dim] = x
    for s in range(len(laid.v)):
        at = (laid.table[s] == p).nonzero()
        if len(at):
            i = int(at[0, 0]) * laid.page + j % laid.page
            if i < laid.lengths[s]:
                laid.v[s][0, i, dim] = x


@pytest.mark.parametrize("shape", [(8, 2, 128), (4, 4, 64), (16, 1, 64)])
def test_not_finite_shared_and_tiles(gpu, shape):
    """Values that are not finite in a shared prefix, in one row's own part, and between the rows of a prompt."""
    per = 11
    laid = pr.Laid([768 + per, 900, 800], shape[1], shape[2], 64, [0, 3], [768], seed=8)
    laid.pool[1][torch.isnan(laid.pool[1])] = math.inf  # what no row sees
    put(laid, 0, 100, 3, math.inf)
    put(laid, 0, 700, 4, math.nan)
    put(laid, 0, 701, 5, -math.inf)
    put(laid, 0, 101, 5, math.inf)  # and its opposite: NaN
    put(laid, 0, 768 + 4, 6, -math.inf)  # seen from the prompt's fifth row on
    put(laid, 1, 800, 7, math.inf)
    tk = [768 + j + 1 for j in range(per)] + [900, 800]
    row = [0] * per + [1, 2]
    got, want, tol, _ = decode(gpu, laid, shape, tk, row, [0, per + 2], [768])
    close(got, want, tol)
    assert torch.isinf(want[5, 0, 6]) and torch.isfinite(want[3, 0, 6]) and torch.isnan(want[0, 0, 5])


def test_not_finite_selected(gpu):
    heads, kv, hd, page, per = 8, 2, 128, 32, 20
    laid = pr.Laid([700], kv, hd, page, seed=8)
    laid.pool[1][torch.isnan(laid.pool[1])] = math.nan
    put(laid, 0, 5 * page + 3, 6, math.inf)
    put(laid, 0, 690, 7, math.nan)
    tk = [700 - per + 1 + j for j in range(per)]
    r = random.Random(1)
    chosen = torch.tensor([[sorted(r.sample(range(21), 5) + [21]) for _ in range(kv)] for _ in range(per)], dtype=torch.int32)
    chosen[3, :, 0], chosen[4, :, 0] = 5, 6
    chosen = chosen.sort(-1).values
    for i in range(per):  # none twice
        for h in range(kv):
            ids = sorted(set(chosen[i, h].tolist()))
            chosen[i, h] = torch.tensor(ids + [-1] * (6 - len(ids)))
    q = queries(3, per, heads, hd)
    got = gpu.attn_decode_selected(q.cuda().view(-1), 0, heads * hd, laid.cache(), ints(laid.table.tolist()), ints([0] * per),
                                   ints(tk), chosen.cuda(), heads, hd ** -0.5)
    want, tol = pr.attend(laid, q, tk, [0] * per, hd ** -0.5, chosen=chosen)
    close(got, want, tol)
    one = gpu.attn_decode_selected(q[3].cuda().view(-1), 0, heads * hd, laid.cache(), ints(laid.table.tolist()), None,
                                   ints(tk[3:4]), chosen[3:4].cuda(), heads, hd ** -0.5)
    close(one, want[3:4], tol[3:4])
    assert torch.isinf(want[3, 0, 6])


@pytest.mark.parametrize("shape", [(8, 2, 128), (2, 2, 64), (32, 2, 64), (5, 1, 128)])
@pytest.mark.parametrize("window", [0, 90])
def test_prompts_rows_masked(gpu, shape, window):
    """Rows of prompts in no group, in tiles that are aligned to sequences and that are not, with windows, caps and
    biases; some rows see nothing."""
    lens = [300, 41, 700]
    laid = pr.Laid(lens, shape[1], shape[2], 32, seed=3)
    per = [37, 41, 64]
    tk = [m - p + 1 + j for m, p in zip(lens, per) for j in range(p)]
    row = [t for t, p in enumerate(per) for _ in range(p)]
    tk[5] = tk[40] = 0
    got, want, tol, plan = decode(gpu, laid, shape, tk, row, window=window, shared=3, softcap=20.0, bias=True, max_tk=700)
    close(got, want, tol)
    assert not got.view(want.shape)[5].any()
    for t, blocks in enumerate(covered(plan, len(tk), shape[0] // shape[1])):
        need = {int(j) // 32 for j in pr.seen_of(tk[t], 0, window, 3, tk[t]).nonzero()}
        assert len(set(blocks)) == len(blocks) and need <= set(blocks)


def test_many_prompt_rows(gpu):
    """More rows than a thread each, of sequences that share a document and of some that do not."""
    shape, per, n = (4, 1, 64), 100, 9
    lens = [256 + per if t < 6 else 90 + per for t in range(n)]
    laid = pr.Laid(lens, 1, 64, 32, [0, 6], [256], seed=3, cols=22)
    tk = [m - per + 1 + j for m in lens for j in range(per)]
    row = [t for t in range(n) for _ in range(per)]
    got, want, tol, plan = decode(gpu, laid, shape, tk, row, [0, 6 * per], [256], max_tk=700)
    close(got, want, tol)
    covered(plan, len(tk), 4)


@pytest.mark.parametrize("shape", [(8, 2, 128), (2, 2, 64), (16, 1, 64)])
@pytest.mark.parametrize("shared", [0, 40])
def test_page_that_later_rows_lack(gpu, shape, shared):
    """Rows of one sequence attended together, of which some need a page that is not there: the others do without it."""
    heads, kv, hd = shape
    page, lens, per = 32, [300, 200], [40, 30]
    laid = pr.Laid(lens, kv, hd, page, seed=3)
    tk = [m - p + 1 + j for m, p in zip(lens, per) for j in range(p)]
    row = [t for t, p in enumerate(per) for _ in range(p)]
    q = queries(5, len(tk), heads, hd)
    table = laid.table.clone()
    table[0, 9] = -1              # positions from 288 on
    table[1, 3] = laid.pages + 7  # from 96 to 127: within a window of some rows
    window = 90
    cache, dt = laid.cache(), ints(table.tolist())
    plan = gpu.page_plan(ints(tk), ints(row), dt, heads, cache, 300, window=window, shared=shared)
    got = gpu.attn_decode_paged(q.cuda().view(-1), 0, heads * hd, cache, plan, heads, hd ** -0.5).view(q.shape).cpu()
    want, tol = pr.attend(laid, q, tk, row, hd ** -0.5, window=window, shared=shared)
    bad = torch.tensor([any(int(j) // page == (9, 3)[t] for j in pr.seen_of(m, 0, window, shared, m).nonzero())
                        for m, t in zip(tk, row)])
    assert 0 < bad.sum() < len(tk)
    assert torch.isnan(got[bad]).all()
    close(got[~bad].contiguous(), want[~bad], tol[~bad])
    # Selected: the even rows choose the pages that are not there.
    chosen = torch.full((len(tk), kv, 4), -1, dtype=torch.int32)
    for r, t in enumerate(row):
        chosen[r] = torch.tensor([0, 2, 4, (9, 3)[t] if r % 2 == 0 else 5], dtype=torch.int32)
    got = gpu.attn_decode_selected(q.cuda().view(-1), 0, heads * hd, cache, dt, ints(row), ints(tk), chosen.cuda(), heads,
                                   hd ** -0.5).view(q.shape).cpu()
    want, tol = pr.attend(laid, q, tk, row, hd ** -0.5, chosen=chosen)
    bad = torch.tensor([r % 2 == 0 and tk[r] > 32 * (9, 3)[t] for r, t in enumerate(row)])
    assert 0 < bad.sum() < len(tk)
    assert torch.isnan(got[bad]).all()
    close(got[~bad].contiguous(), want[~bad], tol[~bad])


def test_more_prompt_rows_than_threads(gpu):
    """Rows of prompts of which a plan's thread takes several, behind shared documents and not."""
    shape, per, n = (4, 2, 64), 130, 9
    lens = [256 + per if t < 3 else 96 + per if t < 5 else 20 + per for t in range(n)]
    laid = pr.Laid(lens, 2, 64, 32, [0, 3, 5], [256, 64], seed=3, cols=13)
    tk = [m - per + 1 + j for m in lens for j in range(per)]
    row = [t for t in range(n) for _ in range(per)]
    got, want, tol, plan = decode(gpu, laid, shape, tk, row, [0, 3 * per, 5 * per], [256, 64], max_tk=400)
    close(got, want, tol)
    covered(plan, len(tk), 2)


@pytest.mark.parametrize("n", [7400, 8192])
def test_select_of_most_held_pages(gpu, n):
    """As many pages as one workgroup holds the scores of."""
    heads, kv, hd, page, units, count = 4, 2, 128, 32, 64, 40
    g = torch.Generator().manual_seed(n)
    mid, half = torch.randn(n, kv, 1, hd, generator=g), 1.0 + torch.randn(n, kv, 1, hd, generator=g).abs()
    bounds = torch.cat([mid + half, mid - half], 2).to(torch.float16)
    table = torch.randperm(n, generator=g)[None].expand(units, -1)
    tk = [n * page - r for r in range(units)]
    q = queries(7, units, heads, hd)
    want = pr.select(q[:1], bounds, table[:1], [0], tk, page, count, 1, 1)
    got = gpu.select_pages(q.cuda().view(-1), 0, heads * hd, bounds.cuda(), ints(table.tolist()), None, ints(tk),
                           n * page, heads, page, count, 1, 1)
    assert torch.equal(got[:1].cpu(), want)


def test_prompt_rows_from_a_graph(gpu):
    """Rows of prompts, planned and attended together, over all and over selected pages, replayed as lengths change."""
    heads, kv, hd, page, cols = 8, 2, 128, 64, 20
    laid = pr.Laid([1200, 1100], kv, hd, page, seed=3, cols=cols)
    cache, table = laid.cache(), ints(laid.table.tolist())
    n = 50
    row, tk = ints([0] * n), ints([1] * n)
    q = queries(5, n, heads, hd)
    dq = q.cuda().view(-1)
    chosen = torch.zeros(n, kv, 3, dtype=torch.int32).cuda()

    def step():
        plan = gpu.page_plan(tk, row, table, heads, cache, cols * page, window=500)
        full = gpu.attn_decode_paged(dq, 0, heads * hd, cache, plan, heads, 0.09)
        some = gpu.attn_decode_selected(dq, 0, heads * hd, cache, table, row, tk, chosen, heads, 0.09)
        return full, some

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    r = random.Random(3)
    for i, split in enumerate([50, 0, 23, 1, 40]):
        lengths = [r.randint(0, 1000) + j % 32 if i != 3 else j for j in range(n)]
        rows = [0] * split + [1] * (n - split)
        pages = torch.tensor([[sorted(r.sample(range(max(3, m // page)), 3)) for _ in range(kv)] for m in lengths],
                             dtype=torch.int32)
        tk.copy_(torch.tensor(lengths, dtype=torch.int32))
        row.copy_(torch.tensor(rows, dtype=torch.int32))
        chosen.copy_(pages)
        graph.replay()
        torch.cuda.synchronize()
        close(held[0], *pr.attend(laid, q, lengths, rows, 0.09, window=500))
        close(held[1], *pr.attend(laid, q, lengths, rows, 0.09, chosen=pages))
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("shape,page", [((6, 2, 64), 4096), ((7, 1, 128), 2048), ((33, 11, 64), 32), ((13, 1, 64), 512)])
def test_queries_out_of_step(gpu, shape, page):
    """Queries four bytes off any larger unit, rows far apart, a context in a buffer that the caller holds."""
    heads, kv, hd = shape
    lens = [4500, 37, 4097]
    laid = pr.Laid(lens, kv, hd, page, seed=2)
    cache, table = laid.cache(), ints(laid.table.tolist())
    per = 5
    tk = [max(1, m - per + 1 + j) for m in lens for j in range(per)]
    row = [t for t in range(3) for _ in range(per)]
    q = queries(4, len(tk), heads, hd)
    stride, off = heads * hd + 3, 5
    flat = torch.full((off + stride * len(tk),), math.nan)
    flat[off:].view(len(tk), stride)[:, :heads * hd] = q.view(len(tk), -1)
    flat = flat.cuda()
    n = len(tk) * heads * hd
    out = torch.full((n + 64,), 7.0, device="cuda")
    plan = gpu.page_plan(ints(tk), ints(row), table, heads, cache, 4500)
    got = gpu.attn_decode_paged(flat, off, stride, cache, plan, heads, hd ** -0.5, out=out)
    want, tol = pr.attend(laid, q, tk, row, hd ** -0.5)
    close(got, want, tol)
    assert (out[n:] == 7.0).all()
    live = max((m + page - 1) // page for m in lens)
    chosen = torch.arange(live, dtype=torch.int32).expand(len(tk), kv, -1).contiguous().cuda()
    out.fill_(7.0)
    got = gpu.attn_decode_selected(flat, off, stride, cache, table, ints(row), ints(tk), chosen, heads, hd ** -0.5, out=out)
    close(got, want, tol)
    assert (out[n:] == 7.0).all()
    if live > 1:
        bounds = torch.zeros(laid.pages, kv, 2, hd, dtype=torch.float16).cuda()
        gpu.page_bounds(cache, table, None, None, ints(lens), max(lens), bounds)
        sel = gpu.select_pages(flat, off, stride, bounds, table, ints(row), ints(tk), 4500, heads, page, live - 1, 0, 1)
        want = pr.select(q, bounds.float().cpu(), laid.table, row, tk, page, live - 1, 0, 1)
        assert torch.equal(sel.cpu(), want)


def test_queries_not_finite(gpu):
    """A NaN or an infinity in one row's queries, among rows attended together: that row's heads alone."""
    heads, kv, hd, page = 8, 2, 128, 32
    lens, per = [300, 333], 24
    laid = pr.Laid(lens, kv, hd, page, [0, 2], [256], seed=3)
    cache, table = laid.cache(), ints(laid.table.tolist())
    tk = [m - per + 1 + j for m in lens for j in range(per)]
    row = [t for t in range(2) for _ in range(per)]
    q = queries(5, len(tk), heads, hd)
    odd = q.clone()
    odd[5, 2, 7], odd[30, 6, 0] = math.nan, math.inf
    chosen = torch.arange(8, dtype=torch.int32).expand(len(tk), kv, -1).contiguous()
    rest = torch.ones(len(tk), heads, dtype=torch.bool)
    rest[5, 2] = rest[30, 6] = False
    plan = gpu.page_plan(ints(tk), ints(row), table, heads, cache, 333, starts=ints([0, 48]), prefix=ints([256]))
    a = gpu.attn_decode_paged(odd.cuda().view(-1), 0, heads * hd, cache, plan, heads, 0.09).view(q.shape).cpu()
    b = gpu.attn_decode_selected(odd.cuda().view(-1), 0, heads * hd, cache, table, ints(row), ints(tk), chosen.cuda(), heads,
                                 0.09).view(q.shape).cpu()
    for got, (want, tol) in ((a, pr.attend(laid, q, tk, row, 0.09)), (b, pr.attend(laid, q, tk, row, 0.09, chosen=chosen))):
        assert got[~rest].isnan().all()
        close(got[rest], want[rest], tol[rest])


def test_nothing(gpu):
    """No rows, no pages chosen, no live positions."""
    heads, kv, hd, page = 8, 2, 128, 32
    laid = pr.Laid([100, 64], kv, hd, page, seed=3)
    cache, table = laid.cache(), ints(laid.table.tolist())
    none, q = ints([]), torch.empty(0, device="cuda")
    plan = gpu.page_plan(none, none, table, heads, cache, 100)
    assert gpu.attn_decode_paged(q, 0, heads * hd, cache, plan, heads, 0.09).numel() == 0
    bounds = torch.full((laid.pages, kv, 2, hd), 3.0, dtype=torch.float16, device="cuda")
    gpu.page_bounds(cache, table, none, None, none, 0, bounds)
    gpu.page_bounds(cache, table, None, None, ints([0, 0]), 5, bounds)
    gpu.page_bounds(cache, table, None, ints([100, 64]), ints([100, 64]), 5, bounds)
    assert (bounds == 3.0).all()
    chosen = gpu.select_pages(q, 0, heads * hd, bounds, table, none, none, 100, heads, page, 2)
    assert chosen.shape == (0, kv, 2)
    assert gpu.attn_decode_selected(q, 0, heads * hd, cache, table, none, none, chosen, heads, 0.09).numel() == 0
    q = queries(3, 2, heads, hd).cuda().view(-1)
    chosen = gpu.select_pages(q, 0, heads * hd, bounds, table, None, ints([0, 0]), 100, heads, page, 2)
    assert (chosen == -1).all()
    got = gpu.attn_decode_selected(q, 0, heads * hd, cache, table, None, ints([100, 64]), chosen, heads, 0.09)
    assert not got.any()
    got = gpu.attn_decode_selected(q, 0, heads * hd, cache, table, None, ints([100, 64]), chosen[:, :, :0].contiguous(), heads,
                                   0.09)
    assert not got.any()
    plan = gpu.page_plan(ints([0, 0]), None, table, heads, cache, 100, starts=ints([0, 2]), prefix=ints([64]))
    assert not gpu.attn_decode_paged(q, 0, heads * hd, cache, plan, heads, 0.09).any()


@pytest.mark.parametrize("seed", range(12))
def test_rows_random(gpu, seed):
    """Rows of prompts and single tokens of several sequences, in order or not, some behind a document in groups of any
    bounds: attended, their pages selected, and attended over selected pages."""
    r = random.Random(seed)
    kv, group, hd = r.choice([1, 2, 3, 5]), r.choice([1, 2, 3, 4, 5, 7, 8, 16]), r.choice([64, 128])
    page, n = r.choice([32, 64, 128, 512]), r.choice([1, 2, 3, 6])
    heads, doc = kv * group, r.choice([0, 0, page, 3 * page, 10 * page])
    lens = [doc + r.choice([1, 5, 33, 100, 400, 900]) for _ in range(n)]
    laid = pr.Laid(lens, kv, hd, page, [0, n], [doc], seed=seed, behind=r.choice([-1, 10**6]))
    rows = []
    for t in range(n):
        m = r.choice([1, 1, 3, 8, 20, 50])
        rows += [(t, max(0, lens[t] - m + 1 + j) if r.random() < 0.9 else r.randint(0, lens[t])) for j in range(m)]
    if r.random() < 0.3:
        r.shuffle(rows)
    row, tk = [t for t, _ in rows], [m for _, m in rows]
    starts = prefix = None
    if doc and r.random() < 0.7:
        starts, prefix = [0, len(row)], [r.choice([doc, doc - 1, max(doc - 33, 0)])]
    if doc and r.random() < 0.3 and len(row) > 4:
        starts, prefix = [1, len(row) // 2, len(row) - 1], [doc, doc // 2]
    window, shared = r.choice([0, 0, 40, 300]), r.choice([0, 0, 4, 70])
    lo = [r.randint(0, 200) for _ in row] if r.random() < 0.3 else None
    cap, bias = r.choice([0.0, 30.0]), r.random() < 0.4
    got, want, tol, plan = decode(gpu, laid, (heads, kv, hd), tk, row, starts, prefix, window, shared, lo, cap, bias,
                                  max_tk=max(lens), seed=seed)
    close(got, want, tol)
    covered(plan, len(row), group)
    q = queries(seed, len(row), heads, hd)
    dq, table, cache = q.cuda().view(-1), ints(laid.table.tolist()), laid.cache()
    bounds = torch.zeros(laid.pages, kv, 2, hd, dtype=torch.float16).cuda()
    gpu.page_bounds(cache, table, None, None, ints(lens), max(lens), bounds)
    count = r.randint(1, max((m + page - 1) // page for m in lens))
    first = r.randint(0, count)
    last = r.randint(0, count - first)
    chosen = gpu.select_pages(dq, 0, heads * hd, bounds, table, ints(row), ints(tk), max(lens), heads, page, count, first,
                              last)
    want = pr.select(q[:8], bounds.cpu(), laid.table, row[:8], tk[:8], page, count, first, last)
    assert torch.equal(chosen[:8].cpu(), want)
    sl = slopes_of(heads) if bias else None
    got = gpu.attn_decode_selected(dq, 0, heads * hd, cache, table, ints(row), ints(tk), chosen, heads, hd ** -0.5, cap,
                                   None if sl is None else sl.cuda())
    close(got, *pr.attend(laid, q, tk, row, hd ** -0.5, cap, sl, chosen=chosen.cpu()))


@pytest.mark.parametrize("size", [1.0, 2.0**14, 2.0**20, 2.0**23, 2.0**28])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_large_equal_scores(gpu, size, sign):
    """Scores of `size` (or less it) at some positions and twice it below at the others: the mean of the values there
    (each weight is the same number, whatever the reference is; f32 sums of up to 700 values lose 700 * 2^-24 of the
    largest, 4.2)."""
    heads, kv, hd, page, n, per = 8, 2, 128, 32, 700, 6
    laid = pr.Laid([n], kv, hd, page, seed=3)
    laid.k[0].zero_()
    laid.k[0][:, :, 0] = sign * 64.0 - 128.0  # far below
    laid.k[0][:, 40::3, 0] = sign * 64.0      # the equal ones
    laid.pool[0].zero_()
    for i in range(laid.table.shape[1]):
        m = min(page, n - i * page)
        laid.pool[0, int(laid.table[0, i]), :, :m] = laid.k[0][:, i * page:i * page + m]
    q = torch.zeros(per, heads, hd)
    q[:, :, 0] = 2.0
    cache, table = laid.cache(), ints(laid.table.tolist())
    tk, row = [n - per + 1 + j for j in range(per)], [0] * per
    chosen = torch.arange(22, dtype=torch.int32).expand(per, kv, -1).contiguous().cuda()
    plan = gpu.page_plan(ints(tk), ints(row), table, heads, cache, n)
    scale = size / 128.0 * math.log(2.0)
    a = gpu.attn_decode_paged(q.cuda().view(-1), 0, heads * hd, cache, plan, heads, scale)
    b = gpu.attn_decode_selected(q.cuda().view(-1), 0, heads * hd, cache, table, ints(row), ints(tk), chosen, heads, scale)
    for got in (a, b):
        got = got.view(per, heads, hd).double().cpu()
        for r in range(per):
            for h in range(heads):
                v = laid.v[0][h // 4, :tk[r]].double()
                w = torch.full((tk[r],), 2.0 ** (-2.0 * min(size, 500.0)), dtype=torch.float64)
                w[40::3] = 1.0
                want = (w[:, None] * v).sum(0) / w.sum()
                assert (got[r, h] - want).abs().max() < 700 * 2.0**-24 * 4.2 + (2e-6 if size == 1.0 else 0.0)
