"""Prompts over key ranges with capped scores, by the kernels of two 16-row query
tiles a wave: where a launch has workgroups enough, and where they are asked for."""
import math

import pytest
import torch

import ranges_ref as ref
from test_ranges_gpu import cache_of, close, f16, prompt, slopes_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("kv", [32, 64, 128])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("c", [
    (1024, 0, {}), (1030, 77, dict(starts=[0, 300, 301, 900, 1010], prefix=[100, 1, 599, 20])),
    (1100, 40, dict(window=130, shared=5)), (1024, 0, dict(causal=False)), (1024, 1100, dict(window=700)),
], ids=lambda c: f"{c[0]}+{c[1]}-{'-'.join(c[2])}")
def test_capped_prompt_of_many_workgroups(gpu, kv, hd, c, bias):
    """1024 workgroups of two tiles or more, in each division of 128 heads over a workgroup's waves; some groups of
    heads are compared. Where documents are, one of them holds values that are not finite, and the last rows see
    nothing."""
    rows, past, table = c
    heads, keys = 128, past + rows
    group = heads // kv
    k, v, q = f16(1, 1, kv, keys, hd), f16(2, 1, kv, keys, hd), f16(3, rows, heads, hd, scale=3.0)
    odd = "starts" in table
    if odd:
        k[0, :, past + 299], v[0, :, past + 299], v[0, :, past + 298, ::3] = math.nan, math.nan, -math.inf
    t = {n: torch.tensor(x, dtype=torch.int32).cuda() if isinstance(x, list) else x for n, x in table.items()}
    sl = slopes_of(heads)
    got = gpu.flash_attn_ranges(q.cuda().view(-1), 0, heads * hd, cache_of(k, v), 0, gpu.key_ranges(rows, past, **t), rows,
                                past, heads, 0.1, 5.0, sl.cuda() if bias else None)
    seen = ref.visible(ref.ranges(rows, past, **table), keys)
    part = slice(300, rows) if odd else slice(0, rows)
    kvs = [0, kv // 2 - 1, kv - 1]
    hs = [h for x in kvs for h in range(x * group, x * group + group)]
    want, tol = ref.attend(q[part][:, hs], k[0, kvs], v[0, kvs], seen[part], torch.arange(past, keys)[part], 0.1, 5.0,
                           sl[hs] if bias else None)
    close(got.view(rows, heads, hd)[part][:, hs].contiguous(), want, tol)
    if odd:
        assert torch.isnan(got.view(rows, -1)[299]).all() and not torch.isnan(got.view(rows, -1)[300:]).any()
        assert not got.view(rows, -1)[1010:].any()


@pytest.mark.parametrize("nqt", ["1", "2"])
@pytest.mark.parametrize("softcap,bias", [(30.0, False), (30.0, True), (0.0, True)])
@pytest.mark.parametrize("shape", [(4, 2, 64), (4, 1, 128), (3, 3, 128)])
def test_capped_prompt_under_the_tile_override(gpu, monkeypatch, nqt, softcap, bias, shape):
    monkeypatch.setenv("LLMTIE_PREFILL_NQT", nqt)
    close(*prompt(gpu, 70, 30, shape, {}, softcap, bias)[:3])
    close(*prompt(gpu, 141, 5, shape, dict(starts=[0, 40, 47, 139], prefix=[7, 9, 30]), softcap, bias)[:3])
