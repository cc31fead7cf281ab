"""The workspace of prompts over key ranges, through the C entry point."""
import pytest
import torch

import ranges_ref as ref
from test_ranges_gpu import cache_of, close, f16

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_keys", [0, 1040, 2000])
def test_a_workspace_of_no_floats_is_none(gpu, max_keys):
    """Its address does not matter then: the keys are not cut. With room they are, to the same context within rounding;
    what lies behind the room is left as it was."""
    rows, past, heads, kv, hd = 40, 1000, 8, 2, 64
    keys = past + rows
    k, v, q = f16(1, 1, kv, keys, hd), f16(2, 1, kv, keys, hd), f16(3, rows, heads, hd)
    cache, dq, r = cache_of(k, v), q.cuda().view(-1), gpu.key_ranges(rows, past)
    L = gpu._L
    n = L.llmtie_flash_attn_ranges_workspace(rows, min(max_keys or keys, keys), heads, kv, hd)
    assert n > 0
    ws = torch.full((n + 64,), 7.0, device="cuda")
    want, tol = ref.attend(q, k[0], v[0], ref.visible(ref.ranges(rows, past), keys), torch.arange(past, keys), 0.1)
    got = []
    for at, floats in ((None, 0), (ws.data_ptr(), 0), (ws.data_ptr(), n)):
        out = torch.zeros(rows * heads * hd, dtype=torch.float16, device="cuda")
        assert L.llmtie_flash_attn_ranges_t16(
            gpu._stream(), dq.data_ptr(), dq.numel(), 0, heads * hd, cache.data.data_ptr(), cache.data.numel(), 1, 0,
            r.table.data_ptr(), r.table.numel(), max_keys, out.data_ptr(), out.numel(), rows, past, heads, kv, hd, keys, 0.1,
            0.0, None, 0, at, floats) == 0
        close(out, want, tol, floats)
        if not floats:
            assert (ws == 7.0).all()
        got.append(out)
    assert torch.equal(got[0], got[1]) and (ws[n:] == 7.0).all() and not (ws[:n] == 7.0).all()
