"""The room that a plan of a step over pages is given, against the items that its rows come to, by the plan's
arithmetic one row at a time. Both are the host's: no launch is made."""
import random
import re
from pathlib import Path

import pytest

from test_abi import last
from test_paged_abi import P, select
from ttsxabe_amd import _lib

WIDE, RUNS, SPAN = 32, 4, 4  # columns of a tile, what part of its rows makes one, blocks of an item at least


def cus():
    L = _lib.lib()
    return (L.llmtie_page_plan_len(1, 0, 2**30, 1, 1, 1) - 32) // 16 // 2


def targets(nseq, max_tk, kv):
    most = (nseq * ((max_tk + 31) // 32) + 3) // 4
    return [max(1, min(n * cus() // kv, most)) for n in ((2 if nseq < 16 else 3), 2)]


def room(nseq, groups, max_tk, table_rows, heads, kv):
    """(items of tiles, of rows by themselves) that there is room for in a plan that divides rows."""
    words = _lib.lib().llmtie_page_plan_len(nseq, groups, max_tk, table_rows, heads, kv)
    own = nseq + targets(nseq, max_tk, kv)[0]
    return (words - (16 + 12 * nseq + 15) // 16 * 16) // 16 - own, own


def need(tk, row, starts, prefix, max_tk, group, kv):
    """The same that the rows come to: all see their first tk positions."""
    n, per = len(tk), WIDE // group
    least = max(2, per // RUNS)
    cost = lambda rows: 7 if min(rows, per) * group > 16 else 4  # noqa: E731
    of, shared = [-1] * n, []
    for g, (a, b) in enumerate(zip(starts, starts[1:])):
        of[a:b] = [g] * (b - a)
        blocks = min([prefix[g]] + tk[a:b]) // 32
        shared.append(blocks if b - a >= 2 else 0)
    tiled = sum(-(-(b - a) // per) * s * cost(b - a) for a, b, s in zip(starts, starts[1:], shared) if s)
    work, runs, r = 0, [], 0
    while r < n:
        e = r + 1
        while e < n and e % per and row[e] == row[r] and of[e] == of[r]:
            e += 1
        for a, b in [(r, e)] if e - r >= least else [(x, x + 1) for x in range(r, e)]:
            s = shared[of[a]] if of[a] >= 0 else 0
            blocks = max((m + 31) // 32 for m in tk[a:b]) - s
            runs.append((b - a, blocks, s))
            if b - a > 1:
                tiled += blocks * cost(b - a)
            else:
                work += blocks * 4
        r = e
    t, tt = targets(n, max_tk, kv)
    c = max(-(-(work + tiled) // (tt if tiled > work else t)), 4 * SPAN)
    wide = sum(-(-(b - a) // per) * -(-s * cost(b - a) // c) for a, b, s in zip(starts, starts[1:], shared) if s)
    own = 0
    for rows, blocks, s in runs:
        items = -(-blocks * (cost(rows) if rows > 1 else 4) // c) if blocks else 0 if s else 1
        if rows > 1:
            wide += items
        else:
            own += items
    return wide, own


@pytest.mark.parametrize("group", range(1, 17))
def test_room_of_runs(group):
    """Rows of many sequences, so many of each: also as many as are just attended together."""
    per = WIDE // group
    for run in sorted({1, 2, 3, max(2, per // RUNS), max(2, per // RUNS) + 1, max(1, per - 1), per}):
        for rows in (40, 970, 3000):
            for tk in (100, 4000):
                for kv in (1, 8, 16):
                    n = max(1, rows // run)
                    row = [t for t in range(n) for _ in range(run)]
                    for starts, prefix in ([0], []), ([0, len(row)], [tk // 2]):
                        has = room(len(row), len(prefix), 4000, n, group * kv, kv)
                        asks = need([tk] * len(row), row, starts, prefix, 4000, group, kv)
                        assert asks[0] <= has[0] and asks[1] <= has[1], (run, rows, tk, kv, prefix, asks, has)


@pytest.mark.parametrize("seed", range(20))
def test_room_of_random_rows(seed):
    r = random.Random(seed)
    for _ in range(20):
        group, kv, n, limit = r.randint(1, 16), r.choice([1, 2, 5, 8, 32]), r.randint(1, 300), r.choice([700, 5000, 100000])
        row = [t for t in range(n) for _ in range(r.choice([1, 2, 2, 3, 5, 8, 40]))]
        tk = [r.choice([0, 1, r.randint(1, limit), limit]) for _ in row]
        starts, prefix = [0], []
        if r.random() < 0.6:
            starts = sorted(r.choices(range(len(row) + 1), k=r.randint(2, 30)))
            prefix = [r.randint(0, limit) for _ in starts[1:]]
        has = room(len(row), len(prefix), limit, n, group * kv, kv)
        asks = need(tk, row, starts, prefix, limit, group, kv)
        assert asks[0] <= max(0, has[0]) and asks[1] <= has[1], (group, kv, len(row), prefix, asks, has)


def test_rows_of_a_selection():
    """More workgroups of 1024 threads than a launch (fewer than 2^32 threads) holds are refused by name."""
    room = dict(row=P, heads=1, kv=1, hd=64, q_len=2**62, ws_len=2**62, chosen_len=2**62)
    for n in (2**22, 2**24 - 600):
        assert select(nseq=n, **room) == 4 and list(last().field)[:2] == [n, 2**22 - 1]


def test_parts_of_a_row():
    """A row's parts are no more than its join takes, however long it and the positions that it shares are."""
    text = (Path(_lib.__file__).parent / "csrc" / "paged.h").read_text()
    most = int(re.search(r"PG_PARTS = (\d+);", text).group(1))
    L = _lib.lib()
    for nseq in (1, 2, 15, 16, 40):
        for groups in (0, 1):
            words = L.llmtie_page_plan_len(nseq, groups, 2**30, nseq, 1, 1)
            items = (words - (16 + 12 * nseq + 15) // 16 * 16) // 16
            # (Room for `target` items beside one a row, or one a tile: twice where rows share.)
            target = (items - nseq) if not groups else (items - nseq - nseq // 32 - 1) // 2
            assert target == targets(nseq, 2**30, 1)[0] and target + 2 <= most
        floats = L.llmtie_attn_selected_workspace(nseq, 2**18, 4096, nseq, 1, 1, 64)
        assert floats <= nseq * (most * 66 + 1)
        floats = L.llmtie_attn_selected_workspace(nseq, 2**18, 4096, 1, 1, 1, 64)
        assert floats <= nseq * (most * 66 + 1) + -(-nseq // 32) * most * 32 * 66
