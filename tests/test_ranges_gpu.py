"""Attention over key ranges (prompts and batched single tokens) against the
plain 64-bit form of ranges_ref, whose tolerance counts the roundings."""
import math
import random

import pytest
import torch

import ranges_ref as ref

pytestmark = pytest.mark.gpu


def f16(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g)).to(torch.float16)


def slopes_of(heads):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32)


def cache_of(k, v):
    """Tiled cache on the device from K, V [slots, kv, cap, hd]; what lies past cap in the last block is NaN."""
    from ttsxabe_amd.gpu import TiledCache16
    slots, kv, cap, hd = k.shape
    pad = (-cap) % 32
    nan = torch.full((slots, kv, pad, hd), math.nan, dtype=torch.float16)
    data = ref.tile(torch.cat([k, nan], 2), torch.cat([v, nan], 2))
    return TiledCache16.of(data.cuda(), kv, hd, cap, slots)


def close(got, want, tol, what=""):
    got = got.double().cpu().view(want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    ok = torch.isfinite(want)
    worst = ((got - want).abs()[ok] / tol[ok].clamp(min=1e-30)).max() if ok.any() else torch.tensor(0.0)
    assert worst <= 1.0, (what, float(worst))
    return float(worst)


# ---------------------------------------------------------------- row table

TABLES = [
    dict(rows=1), dict(rows=173, past=5), dict(rows=257, causal=False), dict(rows=64, window=16, shared=3),
    dict(rows=64, past=100, window=1, shared=200), dict(rows=40, causal=False, window=5),
    dict(rows=50, starts=[0, 17, 17, 49], prefix=[4, 9, 100]), dict(rows=50, starts=[3, 20, 41], past=11, shared=11),
    dict(rows=50, starts=[0, 17, 60], causal=False), dict(rows=33, starts=[40, 50]), dict(rows=9, starts=[2]),
    dict(rows=30, prefix=[12], window=6), dict(rows=700, starts=list(range(0, 701, 7)), window=3, shared=2),
    dict(rows=6000, starts=[2 * i for i in range(3001)]), dict(rows=20, window=2**31 - 1, causal=False),
]


@pytest.mark.parametrize("c", TABLES, ids=lambda c: "-".join(f"{k}{v if not isinstance(v, list) else len(v)}" for k, v in c.items()))
def test_row_table(gpu, c):
    c = dict(c)
    want = ref.ranges(**c)
    for name in ("starts", "prefix"):
        if name in c:
            c[name] = torch.tensor(c[name], dtype=torch.int32).cuda()
    got = gpu.key_ranges(**c)
    assert torch.equal(got.table.cpu(), want[:3]) and torch.equal(got.pos.cpu(), want[3])
    assert got.max_keys >= int(ref.visible(want, c.get("past", 0) + c["rows"]).sum(1).max())


# ------------------------------------------------------------------ prompts

PROMPTS = [
    # rows, past, (heads, kv, hd), row table, softcap, bias
    (1, 0, (4, 4, 64), {}, 0.0, False),
    (1, 63, (8, 2, 128), {}, 30.0, True),
    (17, 0, (4, 2, 64), dict(causal=False), 0.0, True),
    (65, 0, (6, 2, 128), {}, 50.0, False),
    (130, 7, (8, 2, 128), {}, 0.0, False),
    (200, 0, (3, 1, 64), dict(starts=[0, 31, 33, 150, 190]), 0.0, True),
    (200, 60, (8, 2, 128), dict(starts=[0, 64, 128, 200], shared=60), 50.0, False),
    (150, 0, (8, 8, 128), dict(starts=[2, 70, 148], prefix=[40, 200]), 30.0, True),
    (300, 129, (8, 2, 64), dict(window=64, shared=4), 0.0, False),
    (90, 0, (10, 2, 128), dict(causal=False, window=9), 0.0, False),
    (40, 700, (8, 2, 128), dict(window=500, shared=33), 50.0, False),
    (33, 900, (4, 4, 64), {}, 0.0, True),
    (5, 2000, (32, 8, 128), {}, 30.0, False),
    (77, 20, (4, 1, 128), dict(starts=[100, 120]), 0.0, False),
]


def prompt(gpu, rows, past, shape, table, softcap, bias, seed=1, k=None, v=None, q=None, parts=(slice(None),)):
    """`parts`: rows whose reference is computed together (a key seen by one of them is in the sums of all)."""
    heads, kv, hd = shape
    keys = past + rows
    cap = keys + 5
    k = f16(seed + 1, 1, kv, cap, hd) if k is None else k
    v = f16(seed + 2, 1, kv, cap, hd) if v is None else v
    q = f16(seed, rows, heads, hd, scale=3.0) if q is None else q
    k[:, :, keys:], v[:, :, keys:] = math.nan, math.nan  # past the live keys
    t = {n: torch.tensor(x, dtype=torch.int32).cuda() if isinstance(x, list) else x for n, x in table.items()}
    r = gpu.key_ranges(rows, past, **t)
    sl = slopes_of(heads) if bias else None
    scale = hd ** -0.5
    got = gpu.flash_attn_ranges(q.cuda().view(-1), 0, heads * hd, cache_of(k, v), 0, r, rows, past, heads, scale, softcap,
                                sl.cuda() if bias else None)
    seen = ref.visible(ref.ranges(rows, past, **table), keys)
    want, tol = torch.zeros(rows, heads, hd, dtype=torch.float64), torch.zeros(rows, heads, hd, dtype=torch.float64)
    at = torch.arange(past, keys)
    for p in parts:
        want[p], tol[p] = ref.attend(q[p], k[0, :, :keys], v[0, :, :keys], seen[p], at[p], scale, softcap, sl)
    return got, want, tol, seen


@pytest.mark.parametrize("c", PROMPTS, ids=lambda c: f"{c[0]}+{c[1]}-{c[2]}-cap{c[4]}-bias{c[5]}")
def test_prompt(gpu, c):
    got, want, tol, seen = prompt(gpu, *c)
    assert got.dtype == torch.float16
    close(got, want, tol)
    if not seen.any(1).all():  # rows that see nothing
        assert torch.equal(got.view(want.shape)[~seen.any(1)].cpu().double(), want[~seen.any(1)])


@pytest.mark.parametrize("seed", range(12))
def test_prompt_random(gpu, seed):
    r = random.Random(seed)
    rows, past = r.randint(1, 260), r.choice([0, r.randint(1, 1200)])
    table = dict(causal=r.random() < 0.7, window=r.choice([0, r.randint(1, 300)]), shared=r.choice([0, past, 3]))
    if r.random() < 0.5:
        n = r.randint(1, min(rows, 6))
        table["starts"] = sorted(r.choices(range(rows + 1), k=n + 1))
        if r.random() < 0.5:
            table["prefix"] = [r.randint(0, rows) for _ in range(n)]
    shape = r.choice([(8, 2, 128), (4, 4, 64), (12, 4, 64), (5, 5, 128), (16, 1, 128)])
    got, want, tol, _ = prompt(gpu, rows, past, shape, table, r.choice([0.0, 20.0]), r.random() < 0.4, seed=10 * seed)
    close(got, want, tol, (rows, past, table, shape))


@pytest.mark.parametrize("kv", [32, 64, 128])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("c", [
    (1024, 0, {}, False), (1030, 77, dict(starts=[0, 300, 301, 900, 1010], prefix=[100, 1, 599, 20]), True),
    (1100, 40, dict(window=130, shared=5), True), (1024, 0, dict(causal=False), True),
], ids=lambda c: f"{c[0]}+{c[1]}-{'-'.join(c[2])}")
def test_prompt_of_many_workgroups(gpu, kv, hd, c):
    """Enough row blocks for two query tiles a wave, in each division of heads over its waves; some groups of heads
    are compared. Where documents are, one of them holds values that are not finite."""
    rows, past, table, bias = c
    heads, keys = 128, past + rows
    group = heads // kv
    k, v, q = f16(1, 1, kv, keys, hd), f16(2, 1, kv, keys, hd), f16(3, rows, heads, hd, scale=3.0)
    odd = "starts" in table
    if odd:
        k[0, :, past + 299], v[0, :, past + 299], v[0, :, past + 298, ::3] = math.nan, math.nan, -math.inf
    t = {n: torch.tensor(x, dtype=torch.int32).cuda() if isinstance(x, list) else x for n, x in table.items()}
    sl = slopes_of(heads)
    got = gpu.flash_attn_ranges(q.cuda().view(-1), 0, heads * hd, cache_of(k, v), 0, gpu.key_ranges(rows, past, **t), rows,
                                past, heads, 0.1, slopes=sl.cuda() if bias else None)
    seen = ref.visible(ref.ranges(rows, past, **table), keys)
    part = slice(300, rows) if odd else slice(0, rows)
    kvs = [0, kv // 2 - 1, kv - 1]
    hs = [h for x in kvs for h in range(x * group, x * group + group)]
    want, tol = ref.attend(q[part][:, hs], k[0, kvs], v[0, kvs], seen[part], torch.arange(past, keys)[part], 0.1,
                           slopes=sl[hs] if bias else None)
    close(got.view(rows, heads, hd)[part][:, hs].contiguous(), want, tol)
    if odd:
        assert torch.isnan(got.view(rows, -1)[299]).all() and not torch.isnan(got.view(rows, -1)[300:]).any()


def test_prompt_rows_of_a_longer_stride_and_odd_offset(gpu):
    """Queries inside wider rows, aligned or not."""
    rows, heads, kv, hd = 37, 8, 2, 128
    q = f16(3, rows, heads, hd)
    k, v = f16(4, 1, kv, rows, hd), f16(5, 1, kv, rows, hd)
    cache = cache_of(k, v)
    want, tol = ref.attend(q, k[0], v[0], ref.visible(ref.ranges(rows), rows), torch.arange(rows), hd ** -0.5)
    for off, stride in ((0, heads * hd + 8), (8, heads * hd + 256), (3, heads * hd + 5)):
        x = torch.full((off + rows * stride,), math.nan, dtype=torch.float16)
        x[off:].view(rows, stride)[:, :heads * hd] = q.view(rows, -1)
        got = gpu.flash_attn_ranges(x.cuda(), off, stride, cache, 0, gpu.key_ranges(rows), rows, 0, heads, hd ** -0.5)
        close(got, want, tol, (off, stride))


@pytest.mark.parametrize("rows,past", [(120, 0), (30, 900)])
@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_what_a_row_does_not_see_may_be_anything(gpu, rows, past, hd):
    """NaN and infinities in the keys and values of one document leave the others' rows as they are; a row that
    sees an infinite value gets what a sum with it is."""
    heads, kv = 8, 2
    cut = past + rows // 2
    starts = [0, rows // 2, rows]
    k, v = f16(6, 1, kv, past + rows + 5, hd), f16(7, 1, kv, past + rows + 5, hd)
    k[0, :, cut - 3], k[0, :, cut - 4, 5] = math.nan, math.inf
    v[0, :, cut - 3], v[0, :, cut - 4, 0:9:2], v[0, :, cut - 5, 1:9:2] = math.nan, math.inf, -math.inf
    half = rows // 2
    apart = slice(0, half - 5), slice(half, rows)  # rows that see none of them
    got, want, tol, _ = prompt(gpu, rows, past, (heads, kv, hd), dict(starts=starts), 0.0, False, k=k.clone(), v=v.clone(),
                               parts=apart)
    got = got.view(rows, heads, hd).double().cpu()
    for part in apart:
        close(got[part], want[part], tol[part])
    assert torch.isnan(got[half - 3:half]).all()  # rows that see the NaN key
    # Finite keys under infinite values: the rows that see them are infinite there, and finite elsewhere.
    k[0, :, cut - 4:cut - 2] = f16(8, kv, 2, hd)
    v[0, :, cut - 3] = f16(9, kv, hd)
    got, want, tol, _ = prompt(gpu, rows, past, (heads, kv, hd), dict(starts=starts), 0.0, False, k=k, v=v, parts=apart)
    got = got.view(rows, heads, hd).double().cpu()
    see = got[half - 4:half]
    assert (see[..., 0:9:2] == math.inf).all() and (see[..., 1:9:2] == -math.inf).all()
    assert torch.isfinite(see[..., 9:]).all() and torch.isfinite(got[:half - 5]).all() and torch.isfinite(got[half:]).all()


def test_prompt_in_another_slot_and_stream(gpu):
    rows, heads, kv, hd = 50, 4, 2, 64
    k, v = f16(1, 3, kv, 64, hd), f16(2, 3, kv, 64, hd)
    q = f16(3, rows, heads, hd)
    cache = cache_of(k, v)
    want, tol = ref.attend(q, k[2, :, :rows], v[2, :, :rows], ref.visible(ref.ranges(rows), rows), torch.arange(rows),
                           hd ** -0.5)
    r, dq = gpu.key_ranges(rows), q.cuda().view(-1)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = gpu.flash_attn_ranges(dq, 0, heads * hd, cache, 2, r, rows, 0, heads, hd ** -0.5)
    s.synchronize()
    close(got, want, tol)


def test_prompt_ranges_past_the_cache_are_clamped(gpu):
    """A table that a caller made: ranges beyond the keys, negative and empty ones."""
    from ttsxabe_amd.gpu import KeyRanges
    rows, heads, kv, hd = 20, 4, 4, 64
    k, v, q = f16(1, 1, kv, rows, hd), f16(2, 1, kv, rows, hd), f16(3, rows, heads, hd)
    t = torch.zeros(3, rows, dtype=torch.int32)
    t[0], t[1], t[2] = -7, -2**31, 2**31 - 1
    t[:, 3] = torch.tensor([2**31 - 1, 0, 0])
    t[:, 4] = torch.tensor([0, 9, 9])
    t[:, 5] = torch.tensor([3, 12, 2])
    t[:, 6] = torch.tensor([0, 2**31 - 1, -2**31])
    got = gpu.flash_attn_ranges(q.cuda().view(-1), 0, heads * hd, cache_of(k, v), 0, KeyRanges(t.cuda()), rows, 0, heads,
                                hd ** -0.5)
    want, tol = ref.attend(q, k[0], v[0], ref.visible(t, rows), torch.arange(rows), hd ** -0.5)
    close(got, want, tol)
    assert not got.view(rows, -1)[4].any() and not got.view(rows, -1)[6].any()


# ------------------------------------------------------------ single tokens

DECODES = [
    # lengths, cap, (heads, kv, hd), window, shared, softcap, bias
    ([1], 40, (4, 4, 64), 0, 0, 0.0, False),
    ([0, 1, 2, 31, 32, 33], 64, (8, 2, 128), 0, 0, 0.0, True),
    ([257, 3, 129], 300, (16, 1, 128), 0, 0, 50.0, False),
    ([300, 40, 900], 1000, (6, 2, 64), 100, 0, 0.0, True),
    ([300, 40, 900, 0], 1000, (8, 2, 128), 64, 70, 30.0, True),
    ([1000, 5], 1100, (4, 4, 128), 33, 1, 0.0, False),
    ([4001], 4100, (32, 8, 128), 0, 0, 50.0, False),
    ([3000, 2000], 3000, (16, 1, 64), 0, 5000, 0.0, False),
]


def decode(gpu, lens, cap, shape, window, shared, softcap, bias, seed=1, slots=None, lo=None, k=None, v=None, max_tk=None,
           scratch=None):
    from ttsxabe_amd.gpu import DecodeScratch
    heads, kv, hd = shape
    n = len(lens)
    r = random.Random(seed)
    slots = r.sample(range(n + 1), n) if slots is None else slots
    k = f16(seed + 1, n + 1, kv, cap, hd) if k is None else k
    v = f16(seed + 2, n + 1, kv, cap, hd) if v is None else v
    for s, t in zip(slots, lens):
        if 0 <= s <= n:
            k[s, :, t:], v[s, :, t:] = math.nan, math.nan
    q = torch.randn(n, heads, hd, generator=torch.Generator().manual_seed(seed)) * 3.0
    sl = slopes_of(heads) if bias else None
    scale = hd ** -0.5
    ints = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    got = gpu.attn_decode_ranges(q.cuda().view(-1), 0, heads * hd, cache_of(k, v), ints(lens), ints(slots),
                                 max_tk or max(max(lens), 1), heads, scale, scratch or DecodeScratch(), lo_dev=ints(lo),
                                 window=window, shared=shared, softcap=softcap, slopes=sl.cuda() if bias else None)
    want = torch.zeros(n, heads, hd, dtype=torch.float64)
    tol = torch.zeros_like(want)
    for i, (s, t) in enumerate(zip(slots, lens)):
        if not 0 <= s <= n:
            want[i] = math.nan
        elif t:
            first = max(lo[i] if lo else 0, t - window if window else 0)
            seen = ref.visible(torch.tensor([[shared], [first], [t]], dtype=torch.int32), t)
            want[i:i + 1], tol[i:i + 1] = ref.attend(q[i:i + 1], k[s, :, :t], v[s, :, :t], seen, torch.tensor([t - 1]),
                                                     scale, softcap, sl, decode=True)
    return got, want, tol


@pytest.mark.parametrize("c", DECODES, ids=lambda c: f"{c[0]}-{c[2]}-w{c[3]}-s{c[4]}-cap{c[5]}-bias{c[6]}")
def test_decode(gpu, c):
    got, want, tol = decode(gpu, *c)
    assert got.dtype == torch.float32
    close(got, want, tol)


@pytest.mark.parametrize("seed", range(12))
def test_decode_random(gpu, seed):
    r = random.Random(100 + seed)
    n, cap = r.randint(1, 9), r.choice([64, 500, 2000])
    lens = [r.randint(0, cap) for _ in range(n)]
    lo = [r.randint(0, cap) for _ in range(n)] if r.random() < 0.4 else None
    shape = r.choice([(8, 2, 128), (4, 4, 64), (12, 4, 64), (5, 5, 128), (16, 1, 128), (32, 8, 128)])
    args = lens, cap, shape, r.choice([0, r.randint(1, cap)]), r.choice([0, 1, 40]), r.choice([0.0, 20.0]), r.random() < 0.4
    got, want, tol = decode(gpu, *args, seed=seed, lo=lo, max_tk=r.choice([max(lens) or 1, cap]))
    close(got, want, tol, (args, lo))


@pytest.mark.parametrize("c", [
    # Batches whose bound is long: several runs a head, streamed loads, lengths that leave runs without blocks.
    ([4096, 1, 700, 0, 2999, 33, 64, 1500, 4000], (32, 8, 128), 0, 0, 50.0, False),
    ([5] * 9, (32, 8, 128), 0, 0, 0.0, False),
    ([4096] * 9, (16, 8, 128), 0, 0, 0.0, True),
    ([3000, 0, 2000, 17, 4096, 4095, 4090, 2, 1000], (8, 8, 64), 2500, 100, 30.0, True),
    ([4096 - 50 * i for i in range(70)], (4, 1, 64), 0, 0, 0.0, False),  # more than 64 sequences
    ([0] * 64 + [4096, 100], (16, 1, 64), 0, 0, 0.0, False),
], ids=lambda c: f"{len(c[0])}-{c[1]}")
def test_decode_of_long_batches(gpu, c):
    lens, shape, window, shared, softcap, bias = c
    n = len(lens)
    slots = list(range(n)) if n < 20 else [i % 8 for i in range(n)]
    if n >= 20:  # sequences that share slots
        got, want, tol = decode_shared(gpu, lens, shape, slots, *(f16(s, 8, shape[1], 4096, shape[2]) for s in (1, 2)))
    else:
        got, want, tol = decode(gpu, lens, 4096, shape, window, shared, softcap, bias, slots=slots, max_tk=4096)
    close(got, want, tol)


def decode_shared(gpu, lens, shape, slots, k, v):
    """Sequences of several lengths over the same slots."""
    from ttsxabe_amd.gpu import DecodeScratch
    heads, kv, hd = shape
    n = len(lens)
    q = torch.randn(n, heads, hd, generator=torch.Generator().manual_seed(5))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    got = gpu.attn_decode_ranges(q.cuda().view(-1), 0, heads * hd, cache_of(k, v), i32(lens), i32(slots), 4096, heads, 0.1,
                                 DecodeScratch())
    want, tol = (torch.zeros(n, heads, hd, dtype=torch.float64) for _ in range(2))
    for i, (s, t) in enumerate(zip(slots, lens)):
        if t:
            want[i:i + 1], tol[i:i + 1] = ref.attend(q[i:i + 1], k[s, :, :t], v[s, :, :t], torch.ones(1, t, dtype=torch.bool),
                                                     torch.tensor([t - 1]), 0.1, decode=True)
    return got, want, tol


def test_decode_padding_and_shared_slots(gpu):
    """A slot out of range is a NaN row; sequences may share a slot; a length past cap is cut to it."""
    got, want, tol = decode(gpu, [20, 30, 25, 25], 40, (8, 2, 128), 0, 0, 0.0, False, slots=[-1, 9, 2, 2])
    close(got, want, tol)
    from ttsxabe_amd.gpu import DecodeScratch
    kv, hd, cap = 2, 64, 70
    k, v, q = f16(1, 1, kv, cap, hd), f16(2, 1, kv, cap, hd), torch.randn(1, 4, hd)
    got = gpu.attn_decode_ranges(q.cuda().view(-1), 0, 4 * hd, cache_of(k, v), torch.tensor([999], dtype=torch.int32).cuda(),
                                 None, 10, 4, 0.1, DecodeScratch())
    want, tol = ref.attend(q, k[0], v[0], torch.ones(1, cap, dtype=torch.bool), torch.tensor([cap - 1]), 0.1, decode=True)
    close(got, want, tol)


def test_decode_what_is_not_seen_may_be_anything(gpu):
    lens, cap, shape = [400, 77], 420, (8, 2, 128)
    k, v = f16(1, 3, 2, cap, 128), f16(2, 3, 2, cap, 128)
    for t in (k, v):
        t[:, :, 6:9], t[:, :, 40] = math.nan, math.inf
    got, want, tol = decode(gpu, lens, cap, shape, 30, 5, 0.0, False, k=k, v=v)
    assert torch.isfinite(want).all()
    close(got, want, tol)


def test_decode_of_many_runs_is_the_same_each_time(gpu):
    from ttsxabe_amd.gpu import DecodeScratch
    scratch = DecodeScratch()
    args = [2500, 100], 2600, (8, 2, 128), 0, 0, 30.0, False
    first, want, tol = decode(gpu, *args, scratch=scratch)
    close(first, want, tol)
    for _ in range(20):
        again, _, _ = decode(gpu, *args, scratch=scratch)
        assert torch.equal(first, again)


def test_decode_captured_follows_its_lengths(gpu):
    """A captured call reads lengths, slots and cache as they are at each replay, beside eager calls of the same
    scratch."""
    from ttsxabe_amd.gpu import DecodeScratch
    heads, kv, hd, cap, n = 8, 2, 128, 1500, 3
    k, v = f16(1, n, kv, cap, hd), f16(2, n, kv, cap, hd)
    cache, scratch = cache_of(k, v), DecodeScratch()
    q = torch.randn(n, heads, hd, generator=torch.Generator().manual_seed(3))
    dq, out = q.cuda().view(-1), torch.zeros(n * heads * hd, device="cuda")
    tk, slot = torch.ones(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")

    def call(o):
        return gpu.attn_decode_ranges(dq, 0, heads * hd, cache, tk, slot, cap, heads, 0.1, scratch, window=900, shared=9,
                                      out=o)
    call(out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out)
    for lens in ([5, 1500, 33], [1100, 0, 64], [901, 902, 1], [1500, 1500, 1500]):
        tk.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, call(torch.empty_like(out)))
        for i, t in enumerate(lens):
            if t:
                seen = ref.visible(torch.tensor([[9], [t - 900], [t]], dtype=torch.int32), t)
                want, tol = ref.attend(q[i:i + 1], k[i, :, :t], v[i, :, :t], seen, torch.tensor([t - 1]), 0.1, decode=True)
                close(got.view(n, heads, hd)[i:i + 1], want, tol)
            else:
                assert not got.view(n, -1)[i].any()


@pytest.mark.parametrize("softcap", [0.25, 2.0, 4.0, 8.0, 200.0])
@pytest.mark.parametrize("shape", [(8, 2, 64), (4, 4, 128)])
def test_decode_scores_on_both_sides_of_the_series(gpu, shape, softcap):
    """Blocks whose scores are all small against the cap, some beyond 0.45 of it, and all beyond."""
    close(*decode(gpu, [700, 33, 1], 700, shape, 0, 0, softcap, False))


@pytest.mark.parametrize("cap", [1500, 6500])
def test_decode_captured_after_a_larger_batch(gpu, cap):
    """One eager call of the largest batch sizes the scratch for smaller ones, whose heads are cut into more runs."""
    from ttsxabe_amd.gpu import DecodeScratch
    heads, kv, hd, slots = 8, 8, 64, 3
    k, v = f16(1, slots, kv, cap, hd), f16(2, slots, kv, cap, hd)
    cache, scratch = cache_of(k, v), DecodeScratch()
    q = torch.randn(100, heads, hd, generator=torch.Generator().manual_seed(3))
    d = q.cuda().view(-1)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    gpu.attn_decode_ranges(d, 0, heads * hd, cache, i32([100] * 100), i32([0] * 100), cap, heads, 0.1, scratch)
    for n in (1, 3, 25, 40):
        for bound in (cap, 1000):
            lens = [min(bound, 300 * (i % 5) + 1) for i in range(n)]
            tk, slot = i32(lens), i32([i % slots for i in range(n)])
            out = torch.zeros(n * heads * hd, device="cuda")
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                gpu.attn_decode_ranges(d, 0, heads * hd, cache, tk, slot, bound, heads, 0.1, scratch, out=out)
            for turn in range(3):
                out.zero_()
                g.replay()
                torch.cuda.synchronize()
                for i in range(n) if turn == 2 else (0, n - 1):
                    want, tol = ref.attend(q[i:i + 1], k[i % slots, :, :lens[i]], v[i % slots, :, :lens[i]],
                                           torch.ones(1, lens[i], dtype=torch.bool), torch.tensor([lens[i] - 1]), 0.1,
                                           decode=True)
                    close(out.view(n, heads, hd)[i:i + 1], want, tol, (n, bound, i))


def test_prompt_captured(gpu):
    """A cut prompt in a graph: its workspace is the graph's own, and two graphs do not share it."""
    rows, past, heads, kv, hd = 40, 1200, 8, 2, 128
    keys = past + rows
    k, v = f16(1, 1, kv, keys, hd), f16(2, 1, kv, keys, hd)
    cache = cache_of(k, v)
    seen = ref.visible(ref.ranges(rows, past), keys)
    graphs = []
    for s in (3, 4):
        q = f16(s, rows, heads, hd)
        dq, r = q.cuda().view(-1), gpu.key_ranges(rows, past)
        gpu.flash_attn_ranges(dq, 0, heads * hd, cache, 0, r, rows, past, heads, 0.1, 20.0)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = gpu.flash_attn_ranges(dq, 0, heads * hd, cache, 0, r, rows, past, heads, 0.1, 20.0)
        graphs.append((g, out, dq, r, *ref.attend(q, k[0], v[0], seen, torch.arange(past, keys), 0.1, 20.0)))
    for _ in range(3):
        for g, out, *_ in graphs:
            out.zero_()
            g.replay()
        torch.cuda.synchronize()
        for _, out, _, _, want, tol in graphs:
            close(out, want, tol)


def test_a_cache_past_32_bits(gpu):
    """Offsets of the last slot of a cache of more than 2^32 bytes."""
    from ttsxabe_amd.gpu import DecodeScratch, TiledCache16
    heads, kv, hd, cap, slots = 4, 4, 128, 8192, 300
    cache = TiledCache16(kv, hd, cap, zero=False, slots=slots)
    assert cache.data.numel() > 2**31
    n = cache.data.numel() // slots
    k, v = f16(1, 1, kv, cap, hd), f16(2, 1, kv, cap, hd)
    cache.data[-n:] = ref.tile(k, v).cuda()
    q = f16(3, 3, heads, hd)
    seen = ref.visible(ref.ranges(3, cap - 3), cap)
    want, tol = ref.attend(q, k[0], v[0], seen, torch.arange(cap - 3, cap), 0.1)
    got = gpu.flash_attn_ranges(q.cuda().view(-1), 0, heads * hd, cache, slots - 1, gpu.key_ranges(3, cap - 3), 3, cap - 3,
                                heads, 0.1)
    close(got, want, tol)
    got = gpu.attn_decode_ranges(q[2:].float().cuda().view(-1), 0, heads * hd, cache,
                                 torch.tensor([cap], dtype=torch.int32).cuda(),
                                 torch.tensor([slots - 1], dtype=torch.int32).cuda(), cap, heads, 0.1, DecodeScratch())
    want, tol = ref.attend(q[2:].float(), k[0], v[0], seen[2:], torch.tensor([cap - 1]), 0.1, decode=True)
    close(got, want, tol)


def test_distances_past_2_to_the_24(gpu):
    """Positions that f32 does not hold: a bias by distance there is that of the same rows near 0."""
    from ttsxabe_amd.gpu import TiledCache16
    heads, hd, rows, base = 4, 64, 43, 2**24 + 960
    cap = base + 96
    cache = TiledCache16(1, hd, cap, zero=False)
    k, v = f16(1, 1, 1, 96, hd), f16(2, 1, 1, 96, hd)
    cache.data[-(96 * hd * 2):] = ref.tile(k, v).cuda()
    q, slopes = f16(3, rows, heads, hd), slopes_of(heads)
    i = torch.arange(96 - rows, 96)
    table = torch.stack([torch.zeros(rows), torch.zeros(rows), (i + 1.0 + torch.arange(rows) % 9).clamp(max=96)]).int()
    want, tol = ref.attend(q, k[0], v[0], ref.visible(table, 96), i, 0.1, 0.0, slopes)
    from ttsxabe_amd.gpu import KeyRanges
    there = table.clone()
    there[1:] += base
    got = gpu.flash_attn_ranges(q.cuda().view(-1), 0, heads * hd, cache, 0, KeyRanges(there.cuda(), None, 96), rows,
                                cap - rows, heads, 0.1, slopes=slopes.cuda())
    close(got, want, tol)


@pytest.mark.parametrize("softcap", [0.0, 7.0])
@pytest.mark.parametrize("scale", [1e-15, 1e12, 1e15])
def test_extreme_scales(gpu, scale, softcap):
    """Every key of a row far below zero, and scores that are all alike. (With distinct integers as products the
    largest score is exactly known: one key has all the weight, or with a cap those of its sign do.)"""
    from ttsxabe_amd.gpu import DecodeScratch
    heads, hd, n = 4, 64, 70
    k, v = torch.zeros(1, 1, n, hd, dtype=torch.float16), f16(2, 1, 1, n, hd)
    k[0, 0, :, 0] = -1.0 - torch.randperm(n, generator=torch.Generator().manual_seed(1)).half()
    q = torch.zeros(n, heads, hd, dtype=torch.float16)
    q[:, :, 0] = 3.0
    want, tol = ref.attend(q, k[0], v[0], ref.visible(ref.ranges(n), n), torch.arange(n), scale, softcap)
    if scale > 1.0:  # products are exact here, the weights 0 and 1 (or, capped, all alike)
        tol = ref.H * 2 * v.double().abs().amax() + 2.0 ** -20 + 0 * tol
    cache = cache_of(k, v)
    got = gpu.flash_attn_ranges(q.cuda().view(-1), 0, heads * hd, cache, 0, gpu.key_ranges(n), n, 0, heads, scale, softcap)
    close(got, want, tol)
    got = gpu.attn_decode_ranges(q[-1:].float().cuda().view(-1), 0, heads * hd, cache,
                                 torch.tensor([n], dtype=torch.int32).cuda(), None, n, heads, scale, DecodeScratch(),
                                 softcap=softcap)
    close(got, want[-1:], tol[-1:])


@pytest.mark.parametrize("nqt", ["1", "2", "4"])
def test_prompt_under_the_tile_override(gpu, monkeypatch, nqt):
    monkeypatch.setenv("LLMTIE_PREFILL_NQT", nqt)
    close(*prompt(gpu, 70, 30, (4, 2, 64), {}, 0.0, False)[:3])


def test_refusals(gpu):
    from ttsxabe_amd.gpu import DecodeScratch, InvalidArgument, SliceOverrun, TiledCache16
    cache = TiledCache16(2, 64, 40)
    q = torch.zeros(10 * 4 * 64, dtype=torch.float16, device="cuda")
    r = gpu.key_ranges(10)
    with pytest.raises(InvalidArgument):
        gpu.flash_attn_ranges(q.float(), 0, 256, cache, 0, r, 10, 0, 4, 0.1)
    with pytest.raises(InvalidArgument):
        gpu.flash_attn_ranges(q, 0, 256, cache, 0, gpu.key_ranges(11), 10, 0, 4, 0.1)
    with pytest.raises(SliceOverrun):
        gpu.flash_attn_ranges(q, 0, 256, cache, 0, gpu.key_ranges(9), 10, 0, 4, 0.1)
    with pytest.raises(InvalidArgument):
        gpu.flash_attn_ranges(q, -1, 256, cache, 0, r, 10, 0, 4, 0.1)
    with pytest.raises(InvalidArgument):
        gpu.flash_attn_ranges(q.cpu(), 0, 256, cache, 0, r, 10, 0, 4, 0.1)
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    with pytest.raises(SliceOverrun):
        gpu.attn_decode_ranges(q.float(), 0, 256, cache, torch.cat([one, one]), one, 40, 4, 0.1, DecodeScratch())
    with pytest.raises(InvalidArgument):
        gpu.attn_decode_ranges(q.float(), 0, 256, cache, one.long(), one, 40, 4, 0.1, DecodeScratch())
    with pytest.raises(InvalidArgument):
        gpu.key_ranges(-1)
