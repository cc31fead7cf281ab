"""One eager call of the most sequences and the largest bound sizes a scratch for
every smaller one that is captured."""
import pytest
import torch

import ranges_ref as ref
from test_ranges_gpu import cache_of, close, f16

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,cap,most,fewer", [
    # Heads past a round of the compute units are two runs up to one and a half of them; the eager batch is past that.
    ((96, 8, 128), 2048, 49, (48, 43, 40, 33)),
    ((60, 4, 128), 3000, 97, (96, 85, 65)),
    ((88, 8, 128), 6000, 49, (48, 33)),
], ids=lambda c: str(c).replace(" ", ""))
def test_batches_past_a_round_are_captured_after_a_larger_one(gpu, shape, cap, most, fewer):
    from ttsxabe_amd.gpu import DecodeScratch
    heads, kv, hd = shape
    k, v = f16(1, 2, kv, cap, hd), f16(2, 2, kv, cap, hd)
    cache, scratch = cache_of(k, v), DecodeScratch()
    q = torch.randn(most, heads, hd, generator=torch.Generator().manual_seed(3))
    dq = q.cuda().view(-1)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    gpu.attn_decode_ranges(dq, 0, heads * hd, cache, i32([100] * most), i32([0] * most), cap, heads, 0.1, scratch)
    for n in fewer:
        lens = [cap - 37 * i % cap for i in range(n)]
        tk, slot = i32(lens), i32([i % 2 for i in range(n)])
        out = torch.zeros(n * heads * hd, device="cuda")
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            gpu.attn_decode_ranges(dq, 0, heads * hd, cache, tk, slot, cap, heads, 0.1, scratch, out=out)
        for _ in range(3):
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            eager = gpu.attn_decode_ranges(dq, 0, heads * hd, cache, tk, slot, cap, heads, 0.1, DecodeScratch())
            assert torch.equal(out, eager)
        hs = slice(0, 2 * heads // kv)
        for i in (0, n - 1):
            want, tol = ref.attend(q[i:i + 1, hs], k[i % 2, :2, :lens[i]], v[i % 2, :2, :lens[i]],
                                   torch.ones(1, lens[i], dtype=torch.bool), torch.tensor([lens[i] - 1]), 0.1, decode=True)
            close(out.view(n, heads, hd)[i:i + 1, hs].contiguous(), want, tol, (n, i))


@pytest.mark.parametrize("shape,caps", [((96, 8, 128), (64, 2100)), ((64, 4, 128), (64, 6200)), ((8, 2, 64), (32, 6200))],
                         ids=lambda c: str(c).replace(" ", ""))
def test_a_capture_needs_room_for_its_own_runs_only(gpu, shape, caps):
    """A call whose partials fit what an eager one of a shorter bound left is captured: the room that an eager call
    takes for other batches is not asked of it."""
    from ttsxabe_amd.gpu import DecodeScratch
    heads, kv, hd = shape
    least, cap = caps
    k, v = f16(1, 1, kv, cap, hd), f16(2, 1, kv, cap, hd)
    cache, scratch = cache_of(k, v), DecodeScratch()
    q = torch.randn(1, heads, hd, generator=torch.Generator().manual_seed(3))
    dq, tk = q.cuda().view(-1), torch.tensor([least], dtype=torch.int32).cuda()
    out = torch.zeros(heads * hd, device="cuda")
    gpu.attn_decode_ranges(dq, 0, heads * hd, cache, tk, None, least, heads, 0.1, scratch)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gpu.attn_decode_ranges(dq, 0, heads * hd, cache, tk, None, cap, heads, 0.1, scratch, out=out)
    hs = slice(0, 2 * heads // kv)
    for n in (cap, least, cap - 5):
        tk.fill_(n)
        g.replay()
        torch.cuda.synchronize()
        want, tol = ref.attend(q[:, hs], k[0, :2, :n], v[0, :2, :n], torch.ones(1, n, dtype=torch.bool),
                               torch.tensor([n - 1]), 0.1, decode=True)
        close(out.view(1, heads, hd)[:, hs].contiguous(), want, tol, n)
