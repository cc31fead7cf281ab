"""Attention with capped, biased and range-masked scores, and the rotary
producers around it, as cases to time.

Kinds (the `kind` of a case):

  ranges    which keys each row of a packed prompt sees: the row table made
            once for all layers from the documents' starts
  rope      rotary positions over the rows of a prompt: half or interleaved
            pairs, part of the head, scaled for a long context, each row at a
            position of its own
  store     the rotation of q and k with the store of k and v into the slots
            of a tiled f16 cache: `rows` sequences' tokens, or a prompt's rows
  prefill   a prompt's attention over the cache, each row over its own keys
            (documents, a window behind shared leading positions, a prefix
            seen by all), scores capped by a tanh or biased by distance
  decode    one token of `nseq` sequences of ragged lengths over their slots,
            the same scores

The cache is the library's tiled f16 layout: blocks of 32 positions, K then V
in the order of the matrix instructions' operands. The plain form reads and
writes it through a permuted view.
"""
import math
import random

import torch

own = False

THETA = 500000.0


def listed():
    return [
        # Three short documents packed into one prompt: the smallest call, all latency.
        dict(name="ranges_3_docs", kind="ranges", rows=173, past=0, docs=3, causal=True, window=0, shared=0,
             prefix=False),
        # A batch of scoring prompts behind one shared system prompt.
        dict(name="ranges_100_docs", kind="ranges", rows=32768, past=517, docs=100, causal=True, window=0, shared=517,
             prefix=True),
        # A chat turn's queries, interleaved pairs as a GGUF checkpoint holds them, read out of the stacked projection.
        dict(name="rope_turn_interleaved", kind="rope", rows=127, heads=32, hd=128, rot=128, pairs="interleaved",
             scaled=False, far=8192, stacked=True),
        # A long prompt's queries far out in an extended context, a quarter of each head left unrotated.
        dict(name="rope_prompt_scaled", kind="rope", rows=8192, heads=32, hd=128, rot=96, pairs="half", scaled=True,
             far=131072, stacked=False),
        # Serving: the tokens of 32 sequences rotated and stored in one call.
        dict(name="store_step_32", kind="store", rows=32, heads=32, kv=8, hd=128, slots=32, cap=2048, rot=128,
             pairs="half", scaled=True, prompt=False),
        # A document as first prompt into its slot.
        dict(name="store_prompt_2k", kind="store", rows=1999, heads=32, kv=8, hd=128, slots=4, cap=4096, rot=128,
             pairs="interleaved", scaled=False, prompt=True),
        # Short questions packed into one pass, heads biased by distance: latency counts.
        dict(name="prefill_packed_bias", kind="prefill", rows=211, past=0, docs=5, heads=20, kv=20, hd=64, causal=True,
             window=0, shared=0, prefix=False, softcap=0.0, bias=True),
        # A turn of a long chat, a window behind four leading positions that every row sees, scores capped.
        dict(name="prefill_turn_window", kind="prefill", rows=173, past=3011, docs=0, heads=32, kv=8, hd=128,
             causal=True, window=2048, shared=4, prefix=False, softcap=50.0, bias=False),
        # The largest prompt: one document whose leading part all its rows see, a padded tail, scores capped.
        dict(name="prefill_8k_prefix", kind="prefill", rows=8192, past=0, docs=1, heads=32, kv=8, hd=128, causal=True,
             window=0, shared=0, prefix=True, softcap=30.0, bias=False),
        # One user: a token after four thousand positions, scores capped.
        dict(name="decode_1", kind="decode", nseq=1, low=4001, high=4001, heads=32, kv=8, hd=128, window=0, shared=0,
             softcap=50.0, bias=False),
        # Eight sequences with a sliding window behind leading positions, multi-head attention, distance bias.
        dict(name="decode_8_window", kind="decode", nseq=8, low=300, high=4000, heads=40, kv=40, hd=128, window=1024,
             shared=16, softcap=0.0, bias=True),
        # Serving at full length: the most bytes a step reads.
        dict(name="decode_32", kind="decode", nseq=32, low=256, high=8192, heads=32, kv=8, hd=128, window=0, shared=0,
             softcap=50.0, bias=False),
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["ranges", "rope", "store", "prefill", "prefill", "prefill", "decode", "decode", "decode"])
    if kind == "ranges":
        rows, past = _log(rng, 20, 32768), rng.choice([0, rng.randint(1, 4000)])
        docs = rng.choice([0, _log(rng, 1, min(100, rows))])
        return dict(kind=kind, rows=rows, past=past, docs=docs, causal=rng.random() < 0.7,
                    window=rng.choice([0, _log(rng, 16, 4096)]), shared=rng.choice([0, past, 4]),
                    prefix=docs > 0 and rng.random() < 0.5)
    heads, kv, hd = rng.choice([(32, 8, 128), (32, 8, 128), (40, 40, 128), (20, 20, 64), (32, 8, 64), (8, 2, 128),
                                (16, 8, 128)])
    pairs, scaled = rng.choice(["half", "interleaved"]), rng.random() < 0.5
    rot = rng.choice([hd, hd, hd // 2, hd * 3 // 4])
    if kind == "rope":
        return dict(kind=kind, rows=_log(rng, 1, 8192 * 32 // max(heads, 32)), heads=heads, hd=hd, rot=rot, pairs=pairs,
                    scaled=scaled, far=rng.choice([8192, 131072]), stacked=rng.random() < 0.5)
    if kind == "store":
        prompt = rng.random() < 0.5
        rows = _log(rng, 1, 4000) if prompt else rng.randint(1, 32)
        return dict(kind=kind, rows=rows, heads=heads, kv=kv, hd=hd, slots=4 if prompt else 32, cap=4096, rot=rot,
                    pairs=pairs, scaled=scaled, prompt=prompt)
    scores = rng.choice([(0.0, False), (30.0, False), (50.0, False), (0.0, True), (50.0, True)])
    if kind == "prefill":
        rows = _log(rng, 2, 4096)
        past = rng.choice([0, _log(rng, 50, 4000)])
        docs = rng.choice([0, 0, _log(rng, 1, min(16, rows))])
        return dict(kind=kind, rows=rows, past=past, docs=docs, heads=heads, kv=kv, hd=hd,
                    causal=rng.random() < 0.8, window=rng.choice([0, 0, _log(rng, 16, 4096)]),
                    shared=rng.choice([0, past, 4]), prefix=docs > 0 and rng.random() < 0.5, softcap=scores[0],
                    bias=scores[1])
    high = _log(rng, 20, 8192 if kv <= 8 else 4000)
    return dict(kind=kind, nseq=_log(rng, 1, 32), low=rng.randint(1, high), high=high, heads=heads, kv=kv, hd=hd,
                window=rng.choice([0, 0, _log(rng, 16, 4096)]), shared=rng.choice([0, 4, 300]), softcap=scores[0],
                bias=scores[1])


# ------------------------------------------------------------------- inputs


def _gen(seed, what=0):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + what) % (1 << 62))


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _starts(c):
    """The documents' first rows, and the row behind the last: ragged, made from the case's sizes. The last rows
    belong to no document, as a padded batch has them."""
    n, docs = c["rows"], c["docs"]
    if not docs:
        return None
    r = random.Random(n * 131 + docs)
    inner = sorted(r.sample(range(1, n), docs - 1)) if n > docs else list(range(1, docs))
    return [0] + inner + [max(n - n // 50, inner[-1] if inner else 1)]


def _prefix(c, starts):
    """How many leading rows of each document all its rows see."""
    if not c["prefix"]:
        return None
    r = random.Random(c["rows"] * 17 + 3)
    return [r.randint(0, max(1, (b - a) // 2)) for a, b in zip(starts, starts[1:])]


def _lengths(c):
    r = random.Random(c["nseq"] * 1009 + c["high"])
    return [r.randint(c["low"], c["high"]) for _ in range(c["nseq"])]


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


def _ints(v):
    return None if v is None else torch.tensor(v, dtype=torch.int32, device="cuda")


def _cap(need):
    """Positions a cache holds for `need`: powers of two from 256."""
    return max(256, 1 << (need - 1).bit_length())


def _slopes(c):
    """A slope a head, a geometric row from 2^(-8 / heads)."""
    if not c["bias"]:
        return None
    h = torch.arange(1, c["heads"] + 1, dtype=torch.float64)
    return (2.0 ** (-8.0 * h / c["heads"])).to(torch.float32).cuda()


def _filled(g, slots, kv, hd, cap):
    """A tiled f16 cache of normal keys and values (every position, live or not)."""
    blocks = (cap + 31) // 32
    return _normal(g, slots * kv * blocks * 64 * hd).to(torch.float16)


def prepare(case, seed):
    c = dict(case)
    g = _gen(seed)
    s = {"c": c}
    if c["kind"] == "ranges":
        starts = _starts(c)
        prefix = _prefix(c, starts)
        if starts is not None:  # other documents, as another batch has them
            r = random.Random(seed)
            inner = sorted(r.sample(range(1, starts[-1]), len(starts) - 2)) if starts[-1] >= len(starts) else starts[1:-1]
            starts = [0] + inner + [starts[-1]]
        c["past"] += seed % 5  # another turn of the conversation
        s |= {"starts": _ints(starts), "prefix": _ints(prefix)}
        return s
    if c["kind"] == "rope":
        width = (c["heads"] + 2 * max(1, c["heads"] // 8) if c["stacked"] else c["heads"]) * c["hd"]
        s["x"] = _normal(g, c["rows"], width)
        s["pos"] = torch.randint(0, c["far"], (c["rows"],), generator=g, device="cuda", dtype=torch.int32)
        s["div"], s["m"] = _freq_div(c)
        return s
    if c["kind"] == "store":
        n, heads, kv, hd = c["rows"], c["heads"], c["kv"], c["hd"]
        s["qkv"] = _normal(g, n, (heads + 2 * kv) * hd)
        if c["prompt"]:
            first = (seed * 7) % (c["cap"] - n + 1)
            s["slot"] = torch.full((n,), seed % c["slots"], dtype=torch.int32, device="cuda")
            s["index"] = torch.arange(first, first + n, dtype=torch.int32, device="cuda")
        else:
            s["slot"] = torch.randperm(c["slots"], generator=g, device="cuda")[:n].to(torch.int32)
            s["index"] = torch.randint(0, c["cap"], (n,), generator=g, device="cuda", dtype=torch.int32)
        s["pos"] = s["index"].clone()
        s["cache"] = _filled(g, c["slots"], kv, hd, c["cap"])
        s["div"], s["m"] = _freq_div(c)
    elif c["kind"] == "prefill":
        starts = _starts(c)
        s["cap"] = _cap(c["past"] + c["rows"])
        s["q"] = (3.0 * _normal(g, c["rows"], c["heads"] * c["hd"])).to(torch.float16)
        s["cache"] = _filled(g, 1, c["kv"], c["hd"], s["cap"])
        s["slopes"] = _slopes(c)
        f, lo, hi, _ = _row_table(c, _ints(starts), _ints(_prefix(c, starts)))
        s["table"] = torch.stack([f, lo, hi]).to(torch.int32)  # made once for all layers
    else:
        s["cap"] = _cap(c["high"])
        s["q"] = 3.0 * _normal(g, c["nseq"], c["heads"] * c["hd"])
        s["cache"] = _filled(g, c["nseq"], c["kv"], c["hd"], s["cap"])
        s["tk"] = _ints(_lengths(c))
        s["slot"] = torch.randperm(c["nseq"], generator=g, device="cuda").to(torch.int32)
        s["slopes"] = _slopes(c)
    if own:  # the handles that such a program keeps
        from ttsxabe_amd.gpu import DecodeScratch, Gpu, KeyRanges, TiledCache16
        s["gpu"] = Gpu(0)
        slots = c.get("slots", c.get("nseq", 1))
        s["tiled"] = TiledCache16.of(s["cache"], c["kv"], c["hd"], s.get("cap", c.get("cap")), slots=slots)
        if c["kind"] == "prefill":
            most = c["past"] + c["rows"]
            most = min(most, c["window"] + c["shared"]) if c["window"] and c["causal"] and not c["prefix"] else most
            s["ranges"] = KeyRanges(s["table"], None, most)
        if c["kind"] == "decode":
            s["scratch"] = DecodeScratch()
    return s


# ------------------------------------------------------------ the plain form


def _row_table(c, starts, prefix):
    """first, lo, hi and the rotary position of each row."""
    n, past, w = c["rows"], c["past"], c["window"]
    r = torch.arange(n, device="cuda")
    i = r + past
    if starts is None:
        s, e, inside = torch.zeros_like(i), torch.full_like(i, past + n), torch.ones_like(i, dtype=torch.bool)
    else:
        b = starts.long()
        d = (r[:, None] >= b[None, :]).sum(1) - 1
        inside = (d >= 0) & (d < len(b) - 1)
        d = d.clamp(0, len(b) - 2)
        s, e = b[d] + past, b[d + 1] + past
    hi = i + 1 if c["causal"] else e
    lo = s
    if w:
        lo = torch.maximum(lo, i - w + 1)
        hi = hi if c["causal"] else torch.minimum(hi, i + w)
    if prefix is not None:
        hi = torch.maximum(hi, torch.minimum(s + prefix.long()[d], e))
    most = i + 1 if c["causal"] else torch.full_like(i, past + n)
    first = most.clamp(max=c["shared"])
    z = torch.zeros_like(i)
    return tuple(torch.where(inside, t, z) for t in (first, lo, hi, i - s))


def _views(cache, slots, kv, hd):
    """The tiled cache as K [slot, kv, block, 4, 2, 4, dims/32, 4, 8] (a position within its block is 8 a + 4 b + c)
    and V [slot, kv, block, 4, 8, dims/16, 16] (8 a + b)."""
    b = cache.view(slots, kv, -1, 2, 32 * hd)
    k = b[:, :, :, 0].view(slots, kv, -1, 2, hd // 32, 4, 4, 4, 8).permute(0, 1, 2, 6, 3, 7, 4, 5, 8)
    v = b[:, :, :, 1].view(slots, kv, -1, hd // 16, 4, 16, 8).permute(0, 1, 2, 4, 6, 3, 5)
    return k, v


def _keys_values(cache, slots, kv, hd, n):
    """K and V [slots, kv, n, hd] in 32 bits."""
    k, v = _views(cache, slots, kv, hd)
    return (k.float().reshape(slots, kv, -1, hd)[:, :, :n].contiguous(),
            v.float().reshape(slots, kv, -1, hd)[:, :, :n].contiguous())


def _angles(pos, div, rot):
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    f = THETA ** (-2.0 * i / rot)
    if div is not None:
        f = f / div.double()
    a = pos.double()[:, None] * f
    return a.cos().float()[:, None, :], a.sin().float()[:, None, :]


def _rotate(x, pos, div, m, rot, pairs):
    """x [rows, heads, dims] rotated in its first `rot` dims."""
    cos, sin = _angles(pos, div, rot)
    r = x[..., :rot]
    if pairs == "half":
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        y = torch.cat([(a * cos - b * sin) * m, (a * sin + b * cos) * m], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack([(a * cos - b * sin) * m, (a * sin + b * cos) * m], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _attend(q, k, v, seen, distance, scale, cap, slopes):
    """q [b, kv, group, rows, hd] over k, v [b, kv, keys, hd]; seen and distance [b, rows, keys]."""
    b, kv, group, rows, hd = q.shape
    sc = torch.matmul(q.reshape(b, kv, group * rows, hd), k.transpose(-1, -2).contiguous())
    sc = sc.view(b, kv, group, rows, -1).mul_(scale)
    if cap:
        sc.div_(cap).tanh_().mul_(cap)
    if slopes is not None:
        sc.sub_(slopes.view(1, kv, group, 1, 1) * distance[:, None, None])
    sc.masked_fill_(~seen[:, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    sc.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = sc.sum(-1, keepdim=True)
    out = torch.matmul(sc.view(b, kv, group * rows, -1), v).view(b, kv, group, rows, hd)
    return torch.where(total > 0, out / total, torch.zeros_like(out))


def _plain(s):
    c = s["c"]
    if c["kind"] == "ranges":
        return [t.to(torch.int32) for t in _row_table(c, s["starts"], s["prefix"])]
    if c["kind"] == "rope":
        x = s["x"][:, :c["heads"] * c["hd"]].view(c["rows"], c["heads"], c["hd"])
        return _rotate(x, s["pos"], s["div"], s["m"], c["rot"], c["pairs"]).reshape(-1)
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    if c["kind"] == "store":
        n = c["rows"]
        x = s["qkv"].view(n, heads + 2 * kv, hd)
        y = _rotate(x[:, :heads + kv], s["pos"], s["div"], s["m"], c["rot"], c["pairs"])
        kview, vview = _views(s["cache"], c["slots"], kv, hd)
        slot, at, w = s["slot"].long(), s["index"].long() // 32, s["index"].long() % 32
        h = torch.arange(kv, device="cuda")
        i = (slot[:, None], h[None], at[:, None])
        kview[(*i, (w // 8)[:, None], (w // 4 % 2)[:, None], (w % 4)[:, None])] = \
            y[:, heads:].to(torch.float16).view(n, kv, hd // 32, 4, 8)
        vview[(*i, (w // 8)[:, None], (w % 8)[:, None])] = x[:, heads + kv:].to(torch.float16).view(n, kv, hd // 16, 16)
        q = y[:, :heads].reshape(-1)  # a prompt's attention reads its queries in 16 bits, a token's in 32
        return {"q": q.to(torch.float16) if c["prompt"] else q, "cache": s["cache"]}
    scale, group = hd ** -0.5, heads // kv
    if c["kind"] == "prefill":
        n, past = c["rows"], c["past"]
        k, v = _keys_values(s["cache"], 1, kv, hd, past + n)
        f, lo, hi = s["table"].long()[:, :, None]
        j = torch.arange(past + n, device="cuda")[None]
        seen = (j < f) | ((j >= lo) & (j < hi))
        dist = (torch.arange(past, past + n, device="cuda")[:, None] - j).abs()
        q = s["q"].float().view(n, kv, group, hd).permute(1, 2, 0, 3)[None]
        out = _attend(q, k, v, seen[None], dist[None], scale, c["softcap"], s["slopes"])
        return out[0].permute(2, 0, 1, 3).reshape(-1).to(torch.float16)
    n, tk = c["nseq"], s["tk"].long()[:, None]
    k, v = _keys_values(s["cache"], n, kv, hd, c["high"])
    k, v = k[s["slot"].long()], v[s["slot"].long()]
    j = torch.arange(c["high"], device="cuda")[None]
    near = j >= tk - c["window"] if c["window"] else j >= 0
    seen = (j < tk) & (near | (j < c["shared"]))
    q = s["q"].view(n, kv, group, 1, hd)
    out = _attend(q, k, v, seen[:, None], (tk - 1 - j).abs()[:, None], scale, c["softcap"], s["slopes"])
    return out.reshape(-1)


def _kernels(s):
    c = s["c"]
    if c["kind"] in ("ranges", "rope"):
        from ttsxabe_amd.gpu import Gpu
        g = Gpu(0)
    else:
        g = s["gpu"]
    if c["kind"] == "ranges":
        r = g.key_ranges(c["rows"], c["past"], s["starts"], s["prefix"], c["causal"], c["window"], c["shared"])
        return [*r.table, r.pos]
    if c["kind"] == "rope":
        out = torch.empty(c["rows"] * c["heads"] * c["hd"], device="cuda")
        g.rope_rows(s["x"], 0, s["x"].shape[1], s["pos"], s["div"], c["rows"], c["heads"], c["hd"], c["rot"], THETA,
                    s["m"], c["pairs"] == "interleaved", out=out)
        return out
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    if c["kind"] == "store":
        q = torch.empty(c["rows"] * heads * hd, dtype=torch.float16 if c["prompt"] else torch.float32, device="cuda")
        x, width = s["qkv"], (heads + 2 * kv) * hd
        g.t16_rope_store(x, 0, x, heads * hd, x, (heads + kv) * hd, width, s["pos"], s["slot"], s["index"], s["div"],
                         c["rows"], heads, c["rot"], THETA, s["m"], c["pairs"] == "interleaved", s["tiled"], q_out=q)
        return {"q": q, "cache": s["cache"]}
    if c["kind"] == "prefill":
        return g.flash_attn_ranges(s["q"], 0, heads * hd, s["tiled"], 0, s["ranges"], c["rows"], c["past"], heads,
                                   hd ** -0.5, c["softcap"], s["slopes"])
    return g.attn_decode_ranges(s["q"], 0, heads * hd, s["tiled"], s["tk"], s["slot"], c["high"], heads, hd ** -0.5,
                                s["scratch"], window=c["window"], shared=c["shared"], softcap=c["softcap"],
                                slopes=s["slopes"])


def run(state):
    return _kernels(state) if own else _plain(state)


# ------------------------------------------------------- the work and the truth


def _seen_ends(c):
    """first, lo and hi of each row of a prompt, counted on the host."""
    starts = _starts(c)
    prefix = _prefix(c, starts)
    n, past, rows = c["rows"], c["past"], []
    d = 0
    for r in range(n):
        i = r + past
        if starts is None:
            s, e = 0, past + n
        else:
            while d + 1 < len(starts) and starts[d + 1] <= r:
                d += 1
            if d + 1 == len(starts):
                rows.append((0, 0, 0))
                continue
            s, e = past + starts[d], past + starts[d + 1]
        lo, hi = s, (i + 1 if c["causal"] else e)
        if c["window"]:
            lo = max(lo, i - c["window"] + 1)
            hi = hi if c["causal"] else min(hi, i + c["window"])
        if prefix is not None:
            hi = max(hi, min(s + prefix[d], e))
        rows.append((min(c["shared"], i + 1 if c["causal"] else past + n), lo, hi))
    return rows


def work(case):
    c = case
    if c["kind"] == "ranges":
        return {"bytes": 16 * c["rows"] + 4 * (c["docs"] + 1) * (2 if c["prefix"] else 1), "flops": 20 * c["rows"]}
    if c["kind"] == "rope":
        n = c["rows"] * c["heads"] * c["hd"]
        return {"bytes": 8 * n + 4 * c["rows"], "flops": 3 * n}
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    if c["kind"] == "store":
        n = c["rows"] * hd
        return {"bytes": n * ((6 if c["prompt"] else 8) * heads + 12 * kv) + 12 * c["rows"],
                "flops": 3 * n * (heads + kv)}
    if c["kind"] == "prefill":
        pairs, keys = 0, c["past"] + c["rows"]
        seen = [(f, max(f, lo), hi) for f, lo, hi in _seen_ends(c)]
        pairs = sum(f + max(0, hi - lo) for f, lo, hi in seen)
        near = min([lo for f, lo, hi in seen if hi > lo] or [0])
        first = max([f for f, lo, hi in seen] or [0])
        read = keys - max(0, near - first)  # what no row sees is not read
        return {"bytes": c["rows"] * heads * hd * 4 + 4 * kv * read * hd + 12 * c["rows"],
                "flops": 4 * hd * heads * pairs}
    keys = 0
    for t in _lengths(c):
        lo = max(0, t - c["window"]) if c["window"] else 0
        keys += t - lo + min(c["shared"], lo)
    return {"bytes": 4 * kv * hd * keys + 8 * c["nseq"] * heads * hd, "flops": 4 * hd * heads * keys}


def exact(case, seed):
    """The definitions in 64 bits, row by row or head by head."""
    c = dict(case)
    s = prepare(c, seed)
    c = s["c"]
    if c["kind"] == "ranges":
        return None
    f8 = torch.float64

    def turn(x, rot, pairs):
        """x [rows, heads, dims] as complex numbers times m e^(i angle)."""
        i = torch.arange(rot // 2, dtype=f8, device="cuda")
        freq = torch.exp(-2.0 * i / rot * math.log(THETA))
        if s["div"] is not None:
            freq = freq / s["div"].to(f8)
        w = torch.polar(torch.full((x.shape[0], rot // 2), s["m"], dtype=f8, device="cuda"),
                        torch.outer(s["pos"].to(f8), freq))[:, None]
        x = x.to(f8)
        y = x.clone()
        if pairs == "half":
            z = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * w
            y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
        else:
            z = torch.complex(x[..., 0:rot:2].contiguous(), x[..., 1:rot:2].contiguous()) * w
            y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
        return y

    heads, hd = c["heads"], c["hd"]
    if c["kind"] == "rope":
        x = s["x"][:, :heads * hd].reshape(c["rows"], heads, hd)
        return turn(x, c["rot"], c["pairs"]).reshape(-1)
    kv = c["kv"]
    cap = s["cap"] if "cap" in s else c["cap"]
    slots = c.get("slots", c.get("nseq", 1))
    # The halves' places in a block, written out: lane l = 16 g + m holds eight of them.
    e = torch.arange(32 * hd, device="cuda")
    j, m, g = e % 8, e // 8 % 16, e // 128 % 4
    kkey, kdim = 8 * (m // 4) + 4 * (e // (512 * (hd // 32))) + m % 4, 32 * (e // 512 % (hd // 32)) + 8 * g + j
    vkey, vdim = 8 * g + j, 16 * (e // 512) + m
    blocks = s["cache"].view(slots, kv, (cap + 31) // 32, 2, 32 * hd)
    if c["kind"] == "store":
        x = s["qkv"].view(c["rows"], heads + 2 * kv, hd)
        y = turn(x[:, :heads + kv], c["rot"], c["pairs"])
        out = blocks.to(f8)
        k, v = y[:, heads:], x[:, heads + kv:].to(f8)
        for r in range(c["rows"]):
            slot, at = int(s["slot"][r]), int(s["index"][r])
            b = out[slot, :, at // 32]
            b[:, 0, kkey == at % 32] = k[r][:, kdim[kkey == at % 32]]
            b[:, 1, vkey == at % 32] = v[r][:, vdim[vkey == at % 32]]
        return {"q": y[:, :heads].reshape(-1), "cache": out.reshape(-1)}

    def head(slot, h, n):
        k = torch.empty(blocks.shape[2], 32, hd, dtype=f8, device="cuda")
        v = torch.empty_like(k)
        k[:, kkey, kdim] = blocks[slot, h, :, 0].to(f8)
        v[:, vkey, vdim] = blocks[slot, h, :, 1].to(f8)
        return k.view(-1, hd)[:n], v.view(-1, hd)[:n]

    def one(q, k, v, at, seen, slope):
        """q [rows, hd] at positions `at` over k, v [keys, hd]."""
        sc = (q.to(f8) @ k.T) / math.sqrt(hd)
        if c["softcap"]:
            sc = c["softcap"] * torch.tanh(sc / c["softcap"])
        if slope is not None:
            sc = sc - float(slope) * (at[:, None] - torch.arange(len(k), device="cuda")).abs()
        sc = torch.where(seen, sc, -math.inf)
        p = torch.nan_to_num(torch.softmax(sc, -1), nan=0.0) * seen
        return p @ v

    group = heads // kv
    slopes = s["slopes"]
    if c["kind"] == "prefill":
        n, keys = c["rows"], c["past"] + c["rows"]
        ends = torch.tensor(_seen_ends(c), device="cuda")
        j = torch.arange(keys, device="cuda")
        seen = (j < ends[:, :1]) | ((j >= ends[:, 1:2]) & (j < ends[:, 2:]))
        at = torch.arange(c["past"], keys, device="cuda")
        q = s["q"].view(n, heads, hd)
        out = torch.empty(n, heads, hd, dtype=f8, device="cuda")
        for h in range(heads):
            k, v = head(0, h // group, keys)
            out[:, h] = one(q[:, h], k, v, at, seen, None if slopes is None else slopes[h])
        return out.reshape(-1)
    q = s["q"].view(c["nseq"], heads, hd)
    out = torch.empty(c["nseq"], heads, hd, dtype=f8, device="cuda")
    for r, t in enumerate(_lengths(c)):
        j = torch.arange(t, device="cuda")
        seen = (j < c["shared"]) | (j >= t - (c["window"] or t))
        at = torch.tensor([t - 1], device="cuda")
        for h in range(heads):
            if h % group == 0:
                k, v = head(int(s["slot"][r]), h // group, t)
            out[r, h] = one(q[r, h][None], k, v, at, seen[None], None if slopes is None else slopes[h])[0]
    return out.reshape(-1)
