"""A cache in pages, and the operators of a server around it, as cases to time.

Kinds (the `kind` of a case):

  store     the rotation of q and k with the store of k and v where the pages of
            each row's sequence lie: a token of each sequence, or packed prompts
  bounds    the greatest and least key, dim by dim, of the pages that new
            positions lie in: what the choice of pages is made from
  decode    query rows over the pages of their sequences: a token of each, or
            the rows of questions; sequences of a group share the pages of a
            prefix, which is attended once for all of them
  select    the pages of its sequence that each row attends: those whose bounds
            allow the largest product with the heads of a group, the first and
            last ones always
  selected  attention over the pages that were selected for a row and kv head

A page holds a power of two of positions from 32 and is what a slot of the tiled
f16 cache is: per kv head, blocks of 32 positions, K then V in the order of the
matrix instructions' operands. The plain form reads and writes it through a
permuted view. Tables hold the page of each run of positions of a sequence, -1
behind its last.
"""
import math
import random

import torch

own = False

THETA = 500000.0


def listed():
    return [
        # Serving: the tokens of 32 sequences, each into the last page of its own.
        dict(name="store_step_32", kind="store", tables=32, per=1, high=4000, heads=32, kv=8, hd=128, page=64, rot=128,
             pairs="half", scaled=True),
        # Three documents' prompts in one pass, stored page by page.
        dict(name="store_prompts_3", kind="store", tables=3, per=701, high=1003, heads=32, kv=8, hd=128, page=128,
             rot=128, pairs="interleaved", scaled=False),
        # The pages that a step's 32 tokens lie in.
        dict(name="bounds_step_32", kind="bounds", tables=32, per=1, high=4000, kv=8, hd=128, page=64),
        # Four long documents, all their pages.
        dict(name="bounds_prompt_8k", kind="bounds", tables=4, per=0, high=8192, kv=8, hd=128, page=64),
        # Three chats begun behind one short system prompt: all latency.
        dict(name="decode_3", kind="decode", tables=3, per=1, prefix=512, groups=1, low=1, high=60, heads=32, kv=8,
             hd=128, page=64, window=0, shared=0, softcap=0.0, bias=False, plan="kept"),
        # Forty sequences of five customers, some without a prefix, scores capped; the plan made for this call alone.
        dict(name="decode_40_groups", kind="decode", tables=40, per=1, prefix=4096, groups=5, low=20, high=2000,
             heads=32, kv=8, hd=128, page=128, window=0, shared=0, softcap=50.0, bias=False, plan="each"),
        # Questions on one long document: 32 sequences, 8192 positions of them the same.
        dict(name="decode_32_document", kind="decode", tables=32, per=1, prefix=8192, groups=1, low=1, high=300,
             heads=32, kv=8, hd=128, page=64, window=0, shared=0, softcap=0.0, bias=False, plan="kept"),
        # Four questions of 61 tokens read in one pass behind a document of 4096: multi-head attention biased by distance.
        dict(name="decode_4_questions", kind="decode", tables=4, per=61, prefix=4096, groups=1, low=61, high=61,
             heads=20, kv=20, hd=64, page=32, window=0, shared=0, softcap=0.0, bias=True, plan="kept"),
        # One user, 131072 positions: 2048 pages to choose 64 from.
        dict(name="select_1_long", kind="select", tables=1, per=1, low=131001, high=131001, heads=32, kv=8, hd=128,
             page=64, count=64, first=1, last=2),
        # A serving step of 32 sequences in long contexts.
        dict(name="select_32", kind="select", tables=32, per=1, low=2000, high=32768, heads=32, kv=8, hd=128, page=64,
             count=32, first=1, last=2),
        # The same user's attention over the 64 pages.
        dict(name="selected_1_long", kind="selected", tables=1, per=1, low=131001, high=131001, heads=32, kv=8, hd=128,
             page=64, count=64, first=1, last=2, softcap=0.0, bias=False),
        # 127 rows of a prompt, each over 24 pages of its own choice.
        dict(name="selected_rows_127", kind="selected", tables=1, per=127, low=9001, high=9001, heads=32, kv=8, hd=128,
             page=64, count=24, first=1, last=2, softcap=30.0, bias=False),
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["store", "bounds", "decode", "decode", "decode", "select", "select", "selected", "selected"])
    heads, kv, hd = rng.choice([(32, 8, 128), (32, 8, 128), (40, 40, 128), (20, 20, 64), (32, 8, 64), (8, 2, 128),
                                (16, 8, 128), (10, 2, 64), (24, 2, 128)])
    page = rng.choice([32, 64, 64, 128, 256])
    rows = rng.random() < 0.3  # several rows of each sequence
    base = dict(kind=kind, heads=heads, kv=kv, hd=hd, page=page)
    if kind == "store":
        per = _log(rng, 2, 700) if rows else 1
        return base | dict(tables=rng.randint(1, 3 if rows else 32), per=per, high=_log(rng, per + 20, 4000),
                           rot=rng.choice([hd, hd, hd // 2, hd * 3 // 4]), pairs=rng.choice(["half", "interleaved"]),
                           scaled=rng.random() < 0.5)
    if kind == "bounds":
        high = _log(rng, 20, 8192)
        return base | dict(tables=_log(rng, 1, max(1, min(32, 32768 * 8 // (high * kv)))), high=high,
                           per=rng.choice([0, 1, 1, rng.randint(1, high)]))
    scores = rng.choice([(0.0, False), (30.0, False), (50.0, False), (0.0, True), (50.0, True)])
    if kind == "decode":
        prefix = rng.choice([0, _log(rng, 64, 8192), _log(rng, 64, 8192), _log(rng, 64, 8192)])
        per = _log(rng, 2, 64) if rows else 1
        high = max(per, _log(rng, 1, 2000 if prefix else 8192))
        most = max(1, 32 * 8400 * 1024 // ((prefix + high) * kv * hd))
        tables = _log(rng, 1, min(4 if rows else 48, most))
        groups = rng.choice([1, 1, rng.randint(1, min(8, tables))]) if prefix else 0
        return base | dict(tables=tables, per=per, prefix=prefix, groups=groups, low=rng.randint(per, high), high=high,
                           window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), shared=rng.choice([0, 4, 300]),
                           softcap=scores[0], bias=scores[1], plan=rng.choice(["kept", "each"]))
    first, last = rng.randint(0, 2), rng.randint(1, 3)
    per = _log(rng, 2, 100) if rows else 1
    high = _log(rng, 20 * page, 131072 if kind == "select" else 32768)  # longer than what is selected of it
    count = max(first + last + 1, min(high // page // 2, _log(rng, 4, 64)))
    most = max(1, 32 * 16384 * 8 // (high * kv)) if kind == "select" else max(1, 262144 * 1024 // (high * kv * hd))
    tables = _log(rng, 1, max(1, min(2 if rows else 32, most)))
    if kind == "select":  # 64-bit products of the plain form: bounded as the listed ones are
        per = max(1, min(per, 32 * 32768 * 8 // 64 // (tables * kv * (high // page + 1))))
    else:  # no more keys in all than the listed rows have
        count = max(first + last + 1, min(count, 127 * 24 * 64 * 1024 // (tables * per * page * kv * hd)))
    c = base | dict(tables=tables, per=per, low=rng.randint(high // 2, high), high=high, count=count, first=first,
                    last=last)
    return c if kind == "select" else c | dict(softcap=scores[0], bias=scores[1])


# ------------------------------------------------------------------- inputs


def _gen(seed, what=0):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + what) % (1 << 62))


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _lengths(c):
    """Positions of each sequence behind its prefix."""
    r = random.Random(c["tables"] * 1009 + c["high"])
    low = c.get("low", max(1, c["per"]))
    return [r.randint(min(low, c["high"]), c["high"]) for _ in range(c["tables"])]


def _groups(c):
    """First sequence of each group and the one behind the last, and the prefix that each group shares, in whole
    pages: the first group's is the longest, some share nothing."""
    n, groups = c["tables"], c["groups"]
    if not groups:
        return [0, n], [0]
    r = random.Random(n * 131 + groups)
    starts = [0] + sorted(r.sample(range(1, n), groups - 1)) + [n]
    full = max(1, c["prefix"] // c["page"])
    return starts, [c["page"] * (full if i == 0 else r.choice([0, r.randint(1, full)])) for i in range(groups)]


def _ends(c):
    """Live positions of each sequence, and how many of them it shares."""
    own_part = _lengths(c)
    if c["kind"] != "decode":
        return own_part, [0] * c["tables"]
    starts, prefix = _groups(c)
    of = [p for a, b, p in zip(starts, starts[1:], prefix) for _ in range(a, b)]
    return [p + n for p, n in zip(of, own_part)], of


def _tables(c, g):
    """Pages of each sequence [tables, pages of the longest], in no order, and how many pages there are."""
    ends, of = _ends(c)
    page = c["page"]
    wide = max((e + page - 1) // page for e in ends)
    starts = _groups(c)[0] if c["kind"] == "decode" else list(range(c["tables"] + 1))
    ids, n = [], 0
    for a, b in zip(starts, starts[1:]):
        lead = list(range(n, n + of[a] // page))
        n += len(lead)
        for t in range(a, b):
            more = (ends[t] + page - 1) // page - len(lead)
            ids.append(lead + list(range(n, n + more)) + [-1] * (wide - len(lead) - more))
            n += more
    order = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    ids = _ints(ids)
    return torch.where(ids >= 0, order[ids.long().clamp(min=0)], ids), n


def _row_lengths(c):
    """Positions that each query row sees: the last `per` rows of its sequence."""
    return [e - c["per"] + 1 + j for e in _ends(c)[0] for j in range(c["per"])]


def _freq_div(c):
    """Per-frequency divisors of a context extended eightfold: 1 for the fast pairs, 8 for the slow ones, a ramp
    between; and what it multiplies the rotated values by."""
    n = c["rot"] // 2
    if not c["scaled"]:
        return None, 1.0
    i = torch.arange(n, dtype=torch.float64)
    turns = 8192.0 / (2 * math.pi) * THETA ** (-i / n)
    ramp = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
    return (1.0 / (ramp + (1.0 - ramp) / 8.0)).to(torch.float32).cuda(), 1.0 + 0.1 * math.log(8.0)


def _slopes(c):
    """A slope a head, a geometric row from 2^(-8 / heads)."""
    if not c["bias"]:
        return None
    h = torch.arange(1, c["heads"] + 1, dtype=torch.float64)
    return (2.0 ** (-8.0 * h / c["heads"])).to(torch.float32).cuda()


def _chosen(c, g, tk):
    """Pages that rows might have selected, ascending, -1 behind the last: rows of one sequence mostly alike."""
    n, kv, page, count = c["tables"] * c["per"], c["kv"], c["page"], c["count"]
    live = (tk.long() + page - 1) // page
    wide = int((max(_row_lengths(c)) + page - 1) // page)
    like = _normal(g, c["tables"], 1, kv, wide).expand(-1, c["per"], -1, -1).reshape(n, kv, wide)
    like = like + 0.3 * _normal(g, n, kv, wide)
    j = torch.arange(wide, device="cuda")
    kept = (j < c["first"]) | (j >= live[:, None] - c["last"])
    like = like.masked_fill(kept[:, None], math.inf).masked_fill((j >= live[:, None])[:, None], -math.inf)
    top = torch.topk(like, min(count, wide), -1)
    ids = torch.where(top.values > -math.inf, top.indices, wide).sort(-1).values
    ids = torch.where(ids < wide, ids, -1).to(torch.int32)
    return torch.nn.functional.pad(ids, (0, count - ids.shape[-1]), value=-1).contiguous()


def prepare(case, seed):
    c = dict(case)
    g = _gen(seed)
    heads, kv, hd, page = c.get("heads", c["kv"]), c["kv"], c["hd"], c["page"]
    n = c["tables"] * max(1, c["per"])
    s = {"c": c}
    s["table"], pages = _tables(c, g)
    ends = _ends(c)[0]
    s["row"] = torch.arange(c["tables"], dtype=torch.int32, device="cuda").repeat_interleave(max(1, c["per"]))
    if c["kind"] == "bounds":  # of a sequence's positions from `low` on; the whole of it behind a prompt
        s["tk"] = _ints(ends)
        s["low"] = _ints([max(0, e - c["per"]) if c["per"] else 0 for e in ends])
    else:
        s["tk"] = _ints(_row_lengths(c))
    if c["kind"] == "select":  # the bounds of keys, 64 of them or so a page
        mid, half = _normal(g, pages, kv, 1, hd), 2.3 + 0.4 * _normal(g, pages, kv, 1, hd).abs()
        s["bounds"] = torch.cat([0.5 * mid + half, 0.5 * mid - half], 2).to(torch.float16)
    else:
        s["cache"] = _normal(g, pages * kv * page * 2 * hd).to(torch.float16)
    if c["kind"] == "bounds":
        s["bounds"] = torch.zeros(pages, kv, 2, hd, dtype=torch.float16, device="cuda")
    elif c["kind"] == "store":
        s["qkv"] = _normal(g, n, (heads + 2 * kv) * hd)
        s["pos"] = s["tk"] - 1
        s["div"], s["m"] = _freq_div(c)
    else:
        s["q"] = 2.0 * _normal(g, n, heads * hd)
    if c["kind"] == "decode":
        starts, prefix = _groups(c)
        s["starts"], s["prefix"] = _ints([a * c["per"] for a in starts]), _ints(prefix)
    if c["kind"] in ("decode", "selected"):
        s["slopes"] = _slopes(c)
    if c["kind"] == "selected":
        s["chosen"] = _chosen(c, g, s["tk"])
    if own:  # the handles that such a program keeps, and the plan of a step, which serves all layers
        from ttsxabe_amd.gpu import Gpu, PagedCache16
        s["gpu"] = Gpu(0)
        if "cache" in s:
            s["paged"] = PagedCache16.of(s["cache"], kv, hd, pages, page)
        if c.get("plan") == "kept":
            s["plan"] = _plan(s)
    return s


def _plan(s):
    c = s["c"]
    return s["gpu"].page_plan(s["tk"], s["row"], s["table"], c["heads"], s["paged"], s["table"].shape[1] * c["page"],
                              starts=s["starts"], prefix=s["prefix"], window=c["window"], shared=c["shared"])


# ------------------------------------------------------------ the plain form


def _views(cache, kv, hd, page):
    """The pages as K [page, kv, block, 4, 2, 4, dims/32, 4, 8] (a position within its block is 8 a + 4 b + c) and
    V [page, kv, block, 4, 8, dims/16, 16] (8 a + b)."""
    b = cache.view(-1, kv, page // 32, 2, 32 * hd)
    n = b.shape[0]
    k = b[:, :, :, 0].view(n, kv, -1, 2, hd // 32, 4, 4, 4, 8).permute(0, 1, 2, 6, 3, 7, 4, 5, 8)
    v = b[:, :, :, 1].view(n, kv, -1, hd // 16, 4, 16, 8).permute(0, 1, 2, 4, 6, 3, 5)
    return k, v


def _keys_values(s):
    """K and V [page, kv, position, hd] of all pages in 32 bits."""
    c = s["c"]
    k, v = _views(s["cache"], c["kv"], c["hd"], c["page"])
    shape = (-1, c["kv"], c["page"], c["hd"])
    return k.float().reshape(shape), v.float().reshape(shape)


def _attend(q, k, v, at, key, seen, c, slopes):
    """q [b, kv, group, rows, hd] at positions `at` [b, rows] over k, v [b, kv, keys, hd] at positions key [b, kv or 1,
    keys], of which rows see `seen` [b, kv or 1, rows, keys]."""
    b, kv, group, rows, hd = q.shape
    sc = torch.matmul(q.reshape(b, kv, group * rows, hd), k.transpose(-1, -2).contiguous())
    sc = sc.view(b, kv, group, rows, -1).mul_(hd ** -0.5)
    if c["softcap"]:
        sc.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    if slopes is not None:
        sc.sub_(slopes.view(1, kv, group, 1, 1) * (at[:, None, :, None] - key[:, :, None, :]).abs()[:, :, None])
    sc.masked_fill_(~seen[:, :, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    sc.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = sc.sum(-1, keepdim=True)
    out = torch.matmul(sc.view(b, kv, group * rows, -1), v).view(b, kv, group, rows, hd)
    return torch.where(total > 0, out / total, torch.zeros_like(out))


def _rotate(x, pos, div, m, rot, pairs):
    """x [rows, heads, dims] rotated in its first `rot` dims, angles in 64 bits."""
    f = THETA ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64, device="cuda") / rot)
    a = pos.double()[:, None] * (f if div is None else f / div.double())
    cos, sin = a.cos().float()[:, None, :], a.sin().float()[:, None, :]
    r = x[..., :rot]
    if pairs == "half":
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        y = torch.cat([(a * cos - b * sin) * m, (a * sin + b * cos) * m], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack([(a * cos - b * sin) * m, (a * sin + b * cos) * m], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _plain(s):
    c = s["c"]
    kv, hd, page = c["kv"], c["hd"], c["page"]
    tables, per = c["tables"], c["per"]
    tk = s["tk"].long()
    if c["kind"] == "bounds":
        k = _keys_values(s)[0]
        j = torch.arange(s["table"].shape[1] * page, device="cuda").view(1, -1, page)
        live = j < tk[:, None, None]
        first = j[..., 0]
        new = (first < tk[:, None]) & (first + page > s["low"].long()[:, None])
        t, i = new.nonzero(as_tuple=True)
        ids = s["table"][t, i].long()
        off = ~live[t, i][:, None, :, None]
        s["bounds"][ids] = torch.stack([k[ids].masked_fill(off, -math.inf).amax(2),
                                        k[ids].masked_fill(off, math.inf).amin(2)], 2).to(torch.float16)
        return s["bounds"]
    heads, group, n = c["heads"], c["heads"] // kv, tables * per
    row = s["row"].long()
    if c["kind"] == "store":
        x = s["qkv"].view(n, heads + 2 * kv, hd)
        y = _rotate(x[:, :heads + kv], s["pos"], s["div"], s["m"], c["rot"], c["pairs"])
        kview, vview = _views(s["cache"], kv, hd, page)
        at = s["pos"].long()
        ids, b, w = s["table"][row, at // page].long(), at % page // 32, at % 32
        i = (ids[:, None], torch.arange(kv, device="cuda")[None], b[:, None])
        kview[(*i, (w // 8)[:, None], (w // 4 % 2)[:, None], (w % 4)[:, None])] = \
            y[:, heads:].to(torch.float16).view(n, kv, hd // 32, 4, 8)
        vview[(*i, (w // 8)[:, None], (w % 8)[:, None])] = x[:, heads + kv:].to(torch.float16).view(n, kv, hd // 16, 16)
        return {"q": y[:, :heads].reshape(-1), "cache": s["cache"]}
    if c["kind"] == "select":
        b = s["bounds"][s["table"].clamp(min=0).long()].double()  # [tables, pages, kv, 2, hd]
        b = b.permute(0, 2, 4, 3, 1)  # [tables, kv, hd, 2, pages]
        q = s["q"].view(tables, per, kv, group, hd).transpose(1, 2).reshape(tables, kv, per * group, hd).double()
        up = torch.matmul(q.clamp(min=0.0), b[:, :, :, 0].contiguous())
        score = up + torch.matmul(q.clamp(max=0.0), b[:, :, :, 1].contiguous())
        score = score.view(tables, kv, per, group, -1).transpose(1, 2).reshape(n, kv, group, -1)
        score = torch.nan_to_num(score, nan=math.inf, posinf=math.inf, neginf=-math.inf).amax(2)
        live = ((tk + page - 1) // page)[:, None, None]
        j = torch.arange(score.shape[-1], device="cuda")
        score = score.clamp(min=torch.finfo(torch.float64).min)
        score = score.masked_fill((j < c["first"]) | (j >= live - c["last"]), math.inf).masked_fill(j >= live, -math.inf)
        top = torch.sort(score, dim=-1, descending=True, stable=True)
        k = min(c["count"], score.shape[-1])
        ids = torch.where(top.values[..., :k] > -math.inf, top.indices[..., :k], score.shape[-1]).sort(-1).values
        ids = torch.where(ids < score.shape[-1], ids, -1).to(torch.int32)
        return torch.nn.functional.pad(ids, (0, c["count"] - k), value=-1)
    k, v = _keys_values(s)
    if c["kind"] == "decode":
        wide = max(_ends(c)[0])
        ids = s["table"].clamp(min=0).long()
        k, v = (x[ids].transpose(1, 2).reshape(tables, kv, -1, hd)[:, :, :wide] for x in (k, v))
        j = torch.arange(wide, device="cuda")
        t = tk.view(tables, per, 1)
        seen = j < t
        if c["window"]:
            seen = seen & ((j >= t - c["window"]) | (j < c["shared"]))
        q = s["q"].view(tables, per, kv, group, hd).permute(0, 2, 3, 1, 4)
        out = _attend(q, k, v, t[..., 0] - 1, j.view(1, 1, -1), seen[:, None], c, s["slopes"])
        return out.permute(0, 3, 1, 2, 4).reshape(-1)
    page_at = s["chosen"].long().clamp(min=0)  # [n, kv, count]
    ids = s["table"][row[:, None, None], page_at].long().clamp(min=0)
    h = torch.arange(kv, device="cuda")[None, :, None]
    k, v = (x[ids, h].reshape(n, kv, -1, hd) for x in (k, v))
    j = page_at[..., None] * page + torch.arange(page, device="cuda")
    seen = (s["chosen"][..., None] >= 0) & (j < tk[:, None, None, None])
    out = _attend(s["q"].view(n, kv, group, 1, hd), k, v, tk[:, None] - 1, j.flatten(2), seen.flatten(2)[:, :, None], c,
                  s["slopes"])
    return out.reshape(-1)


def _kernels(s):
    c, g = s["c"], s["gpu"]
    if c["kind"] == "bounds":
        g.page_bounds(s["paged"], s["table"], None, s["low"], s["tk"], c["per"] or c["high"], s["bounds"])
        return s["bounds"]
    heads, kv, hd, n = c["heads"], c["kv"], c["hd"], c["tables"] * c["per"]
    if c["kind"] == "store":
        x, width = s["qkv"], (heads + 2 * kv) * hd
        q = torch.empty(n * heads * hd, device="cuda")
        g.paged_rope_store(x, 0, x, heads * hd, x, (heads + kv) * hd, width, s["pos"], s["row"], s["pos"], s["table"],
                           s["div"], n, heads, c["rot"], THETA, s["m"], c["pairs"] == "interleaved", s["paged"], q_out=q)
        return {"q": q, "cache": s["cache"]}
    if c["kind"] == "select":
        return g.select_pages(s["q"], 0, heads * hd, s["bounds"], s["table"], s["row"], s["tk"],
                              s["table"].shape[1] * c["page"], heads, c["page"], c["count"], first=c["first"],
                              last=c["last"])
    if c["kind"] == "decode":
        plan = s["plan"] if c["plan"] == "kept" else _plan(s)
        return g.attn_decode_paged(s["q"], 0, heads * hd, s["paged"], plan, heads, hd ** -0.5, softcap=c["softcap"],
                                   slopes=s["slopes"])
    return g.attn_decode_selected(s["q"], 0, heads * hd, s["paged"], s["table"], s["row"], s["tk"], s["chosen"], heads,
                                  hd ** -0.5, softcap=c["softcap"], slopes=s["slopes"])


def run(state):
    return _kernels(state) if own else _plain(state)


# ------------------------------------------------------- the work and the truth


def _seen(c, t):
    """The leading positions that a row of t positions sees, and the first of the others."""
    lo = max(0, t - c["window"]) if c.get("window") else 0
    return (0, 0) if lo <= c.get("shared", 0) else (min(c["shared"], t), lo)


def work(case):
    c = case
    kv, hd, page = c["kv"], c["hd"], c["page"]
    if c["kind"] == "bounds":
        pages = keys = 0
        for e in _ends(c)[0]:
            first = max(0, e - c["per"]) // page if c["per"] else 0
            keys += e - first * page
            pages += (e + page - 1) // page - first
        return {"bytes": kv * hd * (2 * keys + 4 * pages), "flops": 2 * kv * hd * keys}
    heads, n = c["heads"], c["tables"] * c["per"]
    if c["kind"] == "store":
        return {"bytes": n * (hd * (8 * heads + 12 * kv) + 12), "flops": 3 * n * hd * (heads + kv)}
    ends, of = _ends(c)
    io = 8 * n * heads * hd
    tk = _row_lengths(c)
    if c["kind"] == "select":
        pages = [(t + page - 1) // page for t in tk]
        held = sum((e + page - 1) // page for e in ends)
        return {"bytes": 4 * n * heads * hd + 4 * kv * hd * held + 4 * n * kv * c["count"],
                "flops": 4 * hd * heads * sum(pages)}
    if c["kind"] == "selected":
        keys = [min(t, c["count"] * page - (-t % page)) for t in tk]
        per = [keys[i * c["per"]:(i + 1) * c["per"]] for i in range(c["tables"])]
        read = sum(min(e, sum(k)) for e, k in zip(ends, per))  # rows of one sequence may have chosen the same
        return {"bytes": io + 4 * kv * hd * read + 4 * n * kv * c["count"], "flops": 4 * hd * heads * sum(keys)}
    starts, prefix = _groups(c)
    read = pairs = 0
    for a, b, p in zip(starts, starts[1:], prefix):
        near, first = p, 0
        for t in range(a, b):
            rows = tk[t * c["per"]:(t + 1) * c["per"]]
            seen = [_seen(c, x) for x in rows]
            pairs += sum(f + x - lo for x, (f, lo) in zip(rows, seen))
            low = min(lo for _, lo in seen)
            near, first = min(near, low), max([first] + [f for f, _ in seen])
            read += ends[t] - max(p, low) + max(0, min(first, low) - p)
        read += p - near + min(first, near)
    return {"bytes": io + 4 * kv * hd * read, "flops": 4 * hd * heads * pairs}


def exact(case, seed):
    """The definitions in 64 bits, row by row and head by head."""
    c = dict(case)
    if c["kind"] == "select":
        return None
    s = prepare(c, seed)
    f8 = torch.float64
    kv, hd, page = c["kv"], c["hd"], c["page"]
    # The halves' places in a block, written out: lane l = 16 g + m holds eight of them.
    e = torch.arange(32 * hd, device="cuda")
    j, m, g = e % 8, e // 8 % 16, e // 128 % 4
    kkey, kdim = 8 * (m // 4) + 4 * (e // (512 * (hd // 32))) + m % 4, 32 * (e // 512 % (hd // 32)) + 8 * g + j
    vkey, vdim = 8 * g + j, 16 * (e // 512) + m
    blocks = s["cache"].view(-1, kv, page // 32, 2, 32 * hd)

    def place(ids, h):
        """Keys and values [positions, hd] of pages `ids` of kv head h."""
        b = blocks[ids, h].reshape(-1, 2, 32 * hd)
        k = torch.empty(b.shape[0], 32, hd, dtype=f8, device="cuda")
        v = torch.empty_like(k)
        k[:, kkey, kdim], v[:, vkey, vdim] = b[:, 0].to(f8), b[:, 1].to(f8)
        return k.view(-1, hd), v.view(-1, hd)

    table, ends, tk = s["table"].long(), _ends(c)[0], s["tk"].tolist()
    if c["kind"] == "bounds":
        out = s["bounds"].to(f8)
        for t, end in enumerate(ends):
            first = max(0, end - c["per"]) // page if c["per"] else 0
            for h in range(kv):
                k = place(table[t, first:(end + page - 1) // page], h)[0].view(-1, page, hd)
                at = torch.arange(first * page, first * page + k.shape[0] * page, device="cuda").view(-1, page, 1)
                ids = table[t, first:(end + page - 1) // page]
                out[ids, h, 0] = torch.where(at < end, k, -math.inf).max(1).values
                out[ids, h, 1] = torch.where(at < end, k, math.inf).min(1).values
        return out
    heads, per, n = c["heads"], c["per"], c["tables"] * c["per"]
    if c["kind"] == "store":
        x = s["qkv"].view(n, heads + 2 * kv, hd).to(f8)
        rot = c["rot"]
        freq = torch.exp(-2.0 * torch.arange(rot // 2, dtype=f8, device="cuda") / rot * math.log(THETA))
        if s["div"] is not None:
            freq = freq / s["div"].to(f8)
        w = torch.polar(torch.full((n, rot // 2), s["m"], dtype=f8, device="cuda"), torch.outer(s["pos"].to(f8), freq))
        y = x[:, :heads + kv].clone()
        a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if c["pairs"] == "half" else (slice(0, rot, 2), slice(1, rot, 2))
        z = torch.complex(y[..., a].contiguous(), y[..., b].contiguous()) * w[:, None]
        y[..., a], y[..., b] = z.real, z.imag
        out = blocks.to(f8)
        for r in range(n):
            at = int(s["pos"][r])
            block = out[table[r // per, at // page], :, at % page // 32]
            block[:, 0, kkey == at % 32] = y[r, heads:][:, kdim[kkey == at % 32]]
            block[:, 1, vkey == at % 32] = x[r, heads + kv:][:, vdim[vkey == at % 32]]
        return {"q": y[:, :heads].reshape(-1), "cache": out.reshape(-1)}
    group, slopes = heads // kv, s["slopes"]
    q = s["q"].view(n, heads, hd).to(f8)
    out = torch.zeros(n, heads, hd, dtype=f8, device="cuda")

    def weigh(sc):
        """Scores of products, with the cap."""
        sc = sc / math.sqrt(hd)
        return c["softcap"] * torch.tanh(sc / c["softcap"]) if c["softcap"] else sc

    for t, end in enumerate(ends):
        rows = slice(t * per, (t + 1) * per)
        at = torch.tensor(tk[rows], device="cuda") - 1
        for h in range(kv):
            heads_of = range(h * group, (h + 1) * group)
            if c["kind"] == "decode":
                k, v = (x[:end] for x in place(table[t, :(end + page - 1) // page], h))
                key = torch.arange(end, device="cuda")
                see = torch.zeros(per, end, dtype=torch.bool, device="cuda")
                for i, x in enumerate(tk[rows]):
                    f, lo = _seen(c, x)
                    see[i, :f] = True
                    see[i, lo:x] = True
                for y in heads_of:
                    sc = weigh(q[rows, y] @ k.T)
                    if slopes is not None:
                        sc = sc - float(slopes[y]) * (at[:, None] - key)
                    out[rows, y] = torch.softmax(torch.where(see, sc, -math.inf), -1) @ v
                continue
            for i in range(t * per, (t + 1) * per):
                ids = s["chosen"][i, h].long()
                ids = ids[ids >= 0]
                k, v = place(table[t, ids], h)
                key = (ids[:, None] * page + torch.arange(page, device="cuda")).flatten()
                k, v, key = k[key < tk[i]], v[key < tk[i]], key[key < tk[i]]
                sc = weigh(q[i, h * group:(h + 1) * group] @ k.T)
                if slopes is not None:
                    sc = sc - slopes[h * group:(h + 1) * group, None].to(f8) * (tk[i] - 1 - key)
                out[i, h * group:(h + 1) * group] = torch.softmax(sc, -1) @ v
    return out.reshape(-1)
