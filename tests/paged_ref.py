"""Sequences laid into the pages of a cache, and plain 64-bit forms of what the
paged operators compute (test infrastructure; the attention's error is that of
ranges_ref)."""
import math
import random

import torch

import ranges_ref as ref


class Laid:
    """K, V [sequence][kv, n, hd] (f16) in pages: rows starts[g] to starts[g + 1] of the table hold their first
    prefix[g] positions (whole pages) in the same ones. What no sequence holds is NaN; entries of the table behind
    a sequence's last page are `behind`."""

    def __init__(self, lengths, kv, hd, page, starts=None, prefix=None, seed=0, behind=-1, spare=3, cols=None, scale=1.0):
        g = torch.Generator().manual_seed(seed)
        n = len(lengths)
        starts, prefix = starts or [0, n], prefix or [0]
        self.lengths, self.kv, self.hd, self.page = lengths, kv, hd, page
        self.k, self.v = [], []
        ids, at = [], 0
        fill = []  # (page, sequence, first position)
        need = [(m + page - 1) // page for m in lengths]
        self.cols = cols or max(need + [1])
        group = {t: i for i, (a, b) in enumerate(zip(starts, starts[1:])) for t in range(a, b)}
        lead = {}
        for t, m in enumerate(lengths):
            k = (scale * torch.randn(kv, m, hd, generator=g)).to(torch.float16)
            v = torch.randn(kv, m, hd, generator=g).to(torch.float16)
            row = []
            i = group.get(t)
            if i is not None and prefix[i]:
                p = min(prefix[i], m) // page
                if i not in lead:
                    lead[i] = (list(range(at, at + p)), k[:, :p * page], v[:, :p * page])
                    at += p
                    fill += [(x, t, j * page) for j, x in enumerate(lead[i][0])]
                p = min(p, len(lead[i][0]))
                row = lead[i][0][:p]
                k[:, :p * page], v[:, :p * page] = lead[i][1][:, :p * page], lead[i][2][:, :p * page]
            while len(row) < need[t]:
                fill.append((at, t, len(row) * page))
                row.append(at)
                at += 1
            ids.append(row + [behind] * (self.cols - len(row)))
            self.k.append(k)
            self.v.append(v)
        order = list(range(at + spare))
        random.Random(seed).shuffle(order)
        self.pages = at + spare
        self.table = torch.tensor([[order[x] if 0 <= x < at and x != behind else x for x in r] for r in ids] or
                                  torch.empty(0, self.cols), dtype=torch.int32).view(n, self.cols)
        pool = torch.full((2, self.pages, kv, page, hd), math.nan, dtype=torch.float16)
        for x, t, first in fill:
            m = min(page, lengths[t] - first)
            pool[0, order[x], :, :m] = self.k[t][:, first:first + m]
            pool[1, order[x], :, :m] = self.v[t][:, first:first + m]
        self.pool = pool

    def cache(self):
        from ttsxabe_amd.gpu import PagedCache16
        return PagedCache16.of(ref.tile(self.pool[0], self.pool[1]).cuda(), self.kv, self.hd, self.pages, self.page)


def seen_of(tk, lo, window, shared, n):
    """Positions [n] that a row of tk positions sees."""
    j = torch.arange(n)
    first = max(lo, tk - window if window else 0)
    return (j < tk) & ((j < shared) | (j >= first))


def attend(laid, q, tk, row, scale, softcap=0.0, slopes=None, lo=None, window=0, shared=0, chosen=None):
    """(context, allowed error) of each row: [rows, heads, hd]."""
    want = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros_like(want)
    heads, kv = q.shape[1], laid.kv
    for r in range(len(tk)):
        t, m = row[r], tk[r]
        k, v = laid.k[t][:, :m], laid.v[t][:, :m]
        if m == 0:
            continue
        seen = seen_of(m, lo[r] if lo else 0, window, shared, m)
        for h in range(kv):
            hs = slice(h * (heads // kv), (h + 1) * (heads // kv))
            s = seen
            if chosen is not None:
                pages = {int(x) for x in chosen[r, h] if x >= 0}
                s = torch.tensor([j // laid.page in pages for j in range(m)])
            w, e = ref.attend(q[r:r + 1, hs], k[h:h + 1], v[h:h + 1], s[None], torch.tensor([m - 1]), scale, softcap,
                              None if slopes is None else slopes[hs], decode=True)
            want[r, hs], tol[r, hs] = w[0], e[0]
    return want, tol


def bounds(laid, t, tk, page):
    """Greatest and least key [kv, 2, hd] of page `page` of sequence t, over its positions below tk."""
    k = laid.k[t][:, page * laid.page:min(tk, (page + 1) * laid.page)].float()
    return torch.stack([k.amax(1), k.amin(1)], 1)


def select(q, bounds, table, row, tk, page, count, first, last):
    """[rows, kv, count]: q [rows, heads, hd], bounds [pages, kv, 2, hd]; a page at a time, the sums exactly rounded."""
    rows, heads, hd = q.shape
    kv = bounds.shape[1]
    group = heads // kv
    out = torch.full((rows, kv, count), -1, dtype=torch.int32)
    for r in range(rows):
        t = row[r]
        live = 0 if not 0 <= t < len(table) else (min(tk[r], table.shape[1] * page) + page - 1) // page
        for h in range(kv):
            best = []
            for p in range(live):
                if p < first or p >= live - last:
                    best.append((-math.inf, p))
                    continue
                x = int(table[t, p])
                if not 0 <= x < len(bounds):
                    best.append((-1e308 * 10, p))
                    continue
                b = bounds[x, h].double()
                top = -math.inf
                for y in range(h * group, (h + 1) * group):
                    s = (q[r, y].double().clamp(min=0.0) * b[0] + q[r, y].double().clamp(max=0.0) * b[1]).tolist()
                    s = math.inf if any(math.isnan(z) for z in s) else math.fsum(s) if all(map(math.isfinite, s)) else sum(s)
                    top = max(top, math.inf if math.isnan(s) else s)
                best.append((-top, p))
            forced = [p for p in range(live) if p < first or p >= live - last]
            rest = sorted(b for b in best if b[1] not in set(forced))
            got = sorted(forced + [p for _, p in rest[:max(0, count - len(forced))]])[:count] if live > count else \
                list(range(live))
            out[r, h, :len(got)] = torch.tensor(got, dtype=torch.int32)
    return out
