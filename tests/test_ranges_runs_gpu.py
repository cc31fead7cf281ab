"""Runs of the batched decode over key ranges."""
import torch
import pytest

import ranges_ref as ref
from test_ranges_gpu import cache_of, close, f16

pytestmark = pytest.mark.gpu


def test_batches_around_the_compute_units_agree(gpu):
    """A sequence under a long bound is cut alike whether the batch's heads are some fewer than the compute units, as
    many or some more: its context is the same bits."""
    from ttsxabe_amd.gpu import DecodeScratch
    heads, kv, hd, cap = 16, 8, 128, 6200
    units = torch.cuda.get_device_properties(0).multi_processor_count // kv
    k, v = f16(1, 2, kv, cap, hd), f16(2, 2, kv, cap, hd)
    cache = cache_of(k, v)
    n = units + 1
    q = torch.randn(n, heads, hd, generator=torch.Generator().manual_seed(3))
    dq = q.cuda().view(-1)
    lens = [cap - 97 * i % cap for i in range(n)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    got = [gpu.attn_decode_ranges(dq, 0, heads * hd, cache, i32(lens[:m]), i32([i % 2 for i in range(m)]), cap, heads, 0.1,
                                  DecodeScratch(), softcap=30.0).view(m, heads, hd).cpu() for m in (n - 2, n - 1, n)]
    for g in got:
        assert torch.equal(g[:n - 2], got[0])
    for i in (0, n // 2, n - 1):
        want, tol = ref.attend(q[i:i + 1], k[i % 2, :, :lens[i]], v[i % 2, :, :lens[i]],
                               torch.ones(1, lens[i], dtype=torch.bool), torch.tensor([lens[i] - 1]), 0.1, 30.0, decode=True)
        close(got[-1][i:i + 1], want, tol, i)
