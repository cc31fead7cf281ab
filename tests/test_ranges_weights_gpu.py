"""Rows in which one key has nearly all the weight and many keys a little of it
each: their sum is part of the context, however small each weight is."""
import math

import pytest
import torch

import ranges_ref as ref
from test_ranges_gpu import cache_of, close

pytestmark = pytest.mark.gpu

# Nats of the dominant key above the others: weights of 2^-20.5 and 2^-25.1 of its own.
GAPS = [14.1875, 17.375]


def context(n, at, values, gap, heads, kv, softcap=0.0):
    """(context, tail) of a row over n keys whose scores are `gap` for key `at` and 0 for the others, in 64 bits; `tail`
    the part of the others, of which the weights' errors are a part (the dominant key's own value is 0)."""
    s = torch.zeros(n, dtype=torch.float64)
    s[at] = gap
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    p = torch.softmax(s, 0)
    y = torch.einsum("k,gkd->gd", p, values.double())
    return y.repeat_interleave(heads // kv, 0), float(s[at])


@pytest.mark.parametrize("softcap", [0.0, 100.0])
@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("shape", [(8, 2, 128), (4, 4, 64), (16, 1, 64), (96, 8, 128)])
@pytest.mark.parametrize("n,nseq", [(300, 1), (640, 3), (2000, 48)])
def test_decode_keeps_what_many_small_weights_add(gpu, shape, gap, softcap, n, nseq):
    """Allowed, of the context (all of it the small keys'): their weights' scores, d = 4 u |s| nats and half a step of
    the product with each half of q; 2^-22 and 2^-40 of the largest weight; sums over n keys, u each, of O and of l;
    with a cap the tanh's 16 u c nats."""
    from ttsxabe_amd.gpu import DecodeScratch
    heads, kv, hd = shape
    g = torch.Generator().manual_seed(n)
    at = [0, n // 2, n - 1]
    k = torch.zeros(3, kv, n, hd, dtype=torch.float16)
    v = (1.0 + torch.rand(3, kv, n, hd, generator=g)).to(torch.float16)
    for s in range(3):
        k[s, :, at[s], 3], v[s, :, at[s]] = gap, 0.0
    q = torch.zeros(nseq, heads, hd)
    q[:, :, 3] = 1.0
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    got = gpu.attn_decode_ranges(q.cuda().view(-1), 0, heads * hd, cache_of(k, v), i32([n] * nseq),
                                 i32([i % 3 for i in range(nseq)]), n, heads, 1.0, DecodeScratch(), softcap=softcap)
    got = got.view(nseq, heads, hd).cpu()
    for s in range(min(3, nseq)):
        want, top = context(n, at[s], v[s], gap, heads, kv, softcap)
        small = 2.0 ** -40 * math.exp(top)  # against a small key's weight
        tol = want * (ref.U * (8 * top + 16 * softcap + 4 * n + 8) + 2.0 ** -22 + small)
        for i in range(s, nseq, 3):
            close(got[i], want, tol, (s, i))


@pytest.mark.parametrize("softcap", [0.0, 100.0])
@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("shape", [(128, 1, 128), (256, 1, 64)])
@pytest.mark.parametrize("keys", [2 ** 15, 2 ** 17])
def test_prompts_keep_what_many_small_weights_add(gpu, shape, gap, softcap, keys):
    """Rows enough that no launch cuts the keys: every row's own key, in its first tile, has nearly all the weight, and
    its value is 0. Allowed, of the context (all of it the other keys'): a half step of f16's smallest for each weight,
    2^-25 and as many binades down as the keys are doublings of 2^13, of the largest weight; the scores' 4 u |s| nats,
    the cap's 16 u c; h of each weight and of the output; sums over n keys, u each, of O and of l."""
    heads, kv, hd = shape
    rows = hd
    past = keys - rows
    g = torch.Generator().manual_seed(keys)
    k = torch.zeros(1, kv, keys, hd, dtype=torch.float16)
    v = (1.0 + torch.rand(1, kv, keys, hd, generator=g)).to(torch.float16)
    q = torch.zeros(rows, heads, hd, dtype=torch.float16)
    for r in range(rows):
        q[r, :, r], k[0, 0, past + r, r], v[0, 0, past + r] = 1.0, gap, 0.0
    got = gpu.flash_attn_ranges(q.cuda().view(-1), 0, heads * hd, cache_of(k, v), 0, gpu.key_ranges(rows, past), rows, past,
                                heads, 1.0, softcap)
    top = softcap * math.tanh(gap / softcap) if softcap else gap
    others = torch.arange(past, keys).double()  # keys before a row's own
    want = v[0, 0].double().sum(0)[None] / (math.exp(top) + others[:, None])
    small = 2.0 ** -25 * 2.0 ** 13 / keys * math.exp(top)
    tol = want * (small + 2 * ref.H + ref.U * (8 * top + 16 * softcap + 2 * keys)) + 2.0 ** -25
    got = got.view(rows, heads, hd).cpu()
    for h in (0, heads // 2, heads - 1):
        close(got[:, h].contiguous(), want, tol, h)
    assert torch.equal(got, got[:, :1].expand_as(got))
