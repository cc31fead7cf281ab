"""Rotary positions by row, alone and with the store into a tiled cache, against
the pair-by-pair 64-bit form of ranges_ref.

Tolerance: the sine and cosine are f32's of an angle reduced in f64 (the angle's
half turns are rounded to f32: at most 2^-25 of a half turn, pi 2^-25, and the
functions themselves a few half steps of 1), each times mscale, and a rotated
value is two products and a sum: 16 half steps (2^-24) of mscale (|x| + |y|)
cover them; an f16 output or store adds its half step, 2^-11, and 2^-25."""
import pytest
import torch

import ranges_ref as ref

pytestmark = pytest.mark.gpu
THETA = 500000.0


def rows_of(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def allowed(x, rot, interleaved, m, half):
    """Elementwise: 16 half steps of the pair's magnitude."""
    y = x.double().abs().clone()
    for d in range(rot // 2):
        i, j = (2 * d, 2 * d + 1) if interleaved else (d, d + rot // 2)
        y[..., i] = y[..., j] = x[..., i].double().abs() + x[..., j].double().abs()
    y = 16 * ref.U * abs(m) * y
    y[..., rot:] = 0.0
    want = x.double().abs()
    return y + (ref.H * (abs(m) * 1.42 * want.amax(-1, keepdim=True)) + 2.0 ** -25 if half else 0.0)


CASES = [
    # rows, heads, hd, rot, interleaved, scaled
    (1, 1, 2, 2, False, False), (1, 4, 64, 64, True, False), (3, 5, 128, 128, False, True), (70, 3, 128, 96, True, True),
    (130, 2, 64, 48, False, False), (65, 2, 10, 6, True, False), (9, 1, 36, 20, False, True), (64, 8, 128, 0, False, False),
    (200, 32, 128, 128, False, False), (5, 2, 1024, 1024, True, False),
]


@pytest.mark.parametrize("c", CASES, ids=str)
@pytest.mark.parametrize("to", ["place", "f32", "f16"])
def test_rope_rows(gpu, c, to):
    rows, heads, hd, rot, inter, scaled = c
    x = rows_of(1, rows, heads, hd)
    pos = torch.randint(-3, 200000, (rows,), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    div = 1.0 + rows_of(3, rot // 2).abs() if scaled else None
    m = 1.3 if scaled else 1.0
    want = ref.rotate(x, pos, rot, THETA, div, m, inter)
    d = x.cuda().view(-1)
    out = None if to == "place" else torch.empty(rows * heads * hd, dtype=getattr(torch, "float16" if to == "f16" else "float32"), device="cuda")
    gpu.rope_rows(d, 0, heads * hd, pos.cuda(), div.cuda() if scaled else None, rows, heads, hd, rot, THETA, m, inter, out=out)
    got = (d if out is None else out).double().cpu().view(want.shape)
    assert ((got - want).abs() <= allowed(x, rot, inter, m, to == "f16")).all()
    if to != "f16":
        assert torch.equal(got[..., rot:], x[..., rot:].double())
    if out is not None:
        assert torch.equal(d.cpu(), x.view(-1))


@pytest.mark.parametrize("off,pad", [(0, 0), (4, 12), (3, 5)])
@pytest.mark.parametrize("rows", [7, 90])
def test_rope_rows_inside_wider_rows(gpu, off, pad, rows):
    """In place between other columns, positions from a first one: what lies around stays as it was."""
    heads, hd, rot = 3, 64, 32
    w = heads * hd + pad
    buf = rows_of(4, off + rows * w)
    x = buf[off:].view(rows, w)[:, :heads * hd].reshape(rows, heads, hd)
    d = buf.cuda()
    gpu.rope_rows(d, off, w, 1000, None, rows, heads, hd, rot, THETA)
    want = ref.rotate(x, torch.arange(1000, 1000 + rows), rot, THETA)
    got = d.cpu()[off:].view(rows, w)
    assert ((got[:, :heads * hd].reshape(x.shape).double() - want).abs() <= allowed(x, rot, False, 1.0, False)).all()
    assert torch.equal(got[:, heads * hd:], buf[off:].view(rows, w)[:, heads * hd:]) and torch.equal(d.cpu()[:off], buf[:off])


@pytest.mark.parametrize("rows", [1, 5, 64, 77, 200])
@pytest.mark.parametrize("shape", [(8, 2, 128, 128, False), (4, 4, 64, 48, True), (6, 2, 128, 0, False), (5, 1, 64, 64, False)])
@pytest.mark.parametrize("how", ["scattered", "run", "documents"])
def test_rope_store(gpu, rows, shape, how):
    """Rows into places of all kinds: scattered ones with padding rows, a run from an odd position, documents of
    several slots. The rest of the cache stays as it was."""
    from ttsxabe_amd.gpu import TiledCache16
    heads, kv, hd, rot, inter = shape
    slots, cap = 3, 250
    g = torch.Generator().manual_seed(rows)
    w = (heads + 2 * kv) * hd
    x = torch.randn(rows, w, generator=g)
    pos = torch.randint(0, 100000, (rows,), generator=g, dtype=torch.int32)
    if how == "scattered":
        place = torch.randperm(slots * cap, generator=g)[:rows]
        slot, index = (place // cap).int(), (place % cap).int()
        slot[::5] = torch.tensor([-1, slots])[torch.arange(len(slot[::5])) % 2].int()
        index[3::7] = torch.tensor([-1, cap, 2**31 - 1])[torch.arange(len(index[3::7])) % 3].int()
    elif how == "run":
        slot, index = torch.full((rows,), 1, dtype=torch.int32), torch.arange(13, 13 + rows, dtype=torch.int32)
    else:
        cut = rows // 3
        slot = torch.tensor([2] * cut + [0] * (rows - cut), dtype=torch.int32)
        index = torch.cat([torch.arange(8, 8 + cut), torch.arange(rows - cut)]).int()
    before = ref.tile(*(torch.randn(slots, kv, cap, hd, generator=g).half() for _ in range(2)))
    cache = TiledCache16.of(before.cuda(), kv, hd, cap, slots)
    d, q = x.cuda().view(-1), torch.empty(rows * heads * hd, dtype=torch.float16, device="cuda")
    gpu.t16_rope_store(d, 0, d, heads * hd, d, (heads + kv) * hd, w, pos.cuda(), slot.cuda(), index.cuda(), None, rows,
                       heads, rot, THETA, 1.0, inter, cache, q_out=q)
    assert torch.equal(d.cpu(), x.view(-1))
    x = x.view(rows, heads + 2 * kv, hd)
    want = ref.rotate(x[:, :heads + kv], pos, rot, THETA, interleaved=inter)
    tol = allowed(x[:, :heads + kv], rot, inter, 1.0, True)
    assert ((q.double().cpu().view(rows, heads, hd) - want[:, :heads]).abs() <= tol[:, :heads]).all()
    k0, v0 = ref.untile(before, slots, kv, hd, cap)
    k1, v1 = ref.untile(cache.data.cpu(), slots, kv, hd, cap)
    for r in range(rows):
        s, i = int(slot[r]), int(index[r])
        if 0 <= s < slots and 0 <= i < cap:
            assert ((k1[s, :, i].double() - want[r, heads:]).abs() <= tol[r, heads:]).all(), r
            assert torch.equal(v1[s, :, i], x[r, heads + kv:].half()), r
            k0[s, :, i], v0[s, :, i] = k1[s, :, i], v1[s, :, i]
    assert torch.equal(ref.tile(k0, v0), ref.tile(k1, v1))
    nb = -(-cap // 32) * 32
    assert torch.equal(ref.untile(cache.data.cpu(), slots, kv, hd, nb)[0][:, :, cap:],
                       ref.untile(before, slots, kv, hd, nb)[0][:, :, cap:])


def test_rope_store_in_place_and_without_queries(gpu):
    from ttsxabe_amd.gpu import TiledCache16
    heads, kv, hd, rows = 4, 2, 64, 6
    w = (heads + 2 * kv) * hd
    x = rows_of(5, rows, w)
    at = torch.arange(rows, dtype=torch.int32).cuda()
    zero = torch.zeros_like(at)
    caches = [TiledCache16(kv, hd, 40) for _ in range(2)]
    d = x.cuda().view(-1)
    gpu.t16_rope_store(None, 0, d, heads * hd, d, (heads + kv) * hd, w, at, zero, at, None, rows, heads, hd, THETA, 1.0,
                       False, caches[0])
    assert torch.equal(d.cpu(), x.view(-1))
    gpu.t16_rope_store(d, 0, d, heads * hd, d, (heads + kv) * hd, w, at, zero, at, None, rows, heads, hd, THETA, 1.0, False,
                       caches[1])
    assert torch.equal(caches[0].data, caches[1].data)
    got = d.cpu().view(rows, -1, hd)
    xs = x.view(rows, -1, hd)
    assert ((got[:, :heads].double() - ref.rotate(xs[:, :heads], at.cpu(), hd, THETA)).abs()
            <= allowed(xs[:, :heads], hd, False, 1.0, False)).all()
    assert torch.equal(got[:, heads:], xs[:, heads:])


def test_rope_store_captured(gpu):
    """A captured step follows the positions, slots and rows it reads."""
    from ttsxabe_amd.gpu import TiledCache16
    heads, kv, hd, rows, cap = 8, 2, 128, 3, 64
    w = (heads + 2 * kv) * hd
    cache, again = TiledCache16(kv, hd, cap, slots=rows), TiledCache16(kv, hd, cap, slots=rows)
    x, q, q2 = torch.zeros(rows * w, device="cuda"), *(torch.zeros(rows * heads * hd, device="cuda") for _ in range(2))
    at, slot = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.arange(rows, dtype=torch.int32, device="cuda")

    def call(c, out):
        gpu.t16_rope_store(x, 0, x, heads * hd, x, (heads + kv) * hd, w, at, slot, at, None, rows, heads, hd, THETA, 1.0,
                           True, c, q_out=out)
    call(cache, q)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(cache, q)
    cache.data.zero_()
    for i in range(4):
        x.copy_(rows_of(i, rows * w))
        at.fill_(3 + i)
        g.replay()
        call(again, q2)
        torch.cuda.synchronize()
        assert torch.equal(cache.data, again.data) and torch.equal(q, q2)


def test_refusals(gpu):
    from ttsxabe_amd.gpu import InvalidArgument, SliceOverrun, TiledCache16
    x = torch.zeros(4 * 256, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(InvalidArgument):
        gpu.rope_rows(x.half(), 0, 256, pos, None, 4, 4, 64, 64, THETA)
    with pytest.raises(InvalidArgument):
        gpu.rope_rows(x, 0, 256, pos.long(), None, 4, 4, 64, 64, THETA)
    with pytest.raises(InvalidArgument):
        gpu.rope_rows(x, 0, 256, pos, None, 3, 4, 64, 64, THETA, out=x, out_off=64)
    with pytest.raises(SliceOverrun):
        gpu.rope_rows(x, 1, 256, pos, None, 4, 4, 64, 64, THETA)
    with pytest.raises(SliceOverrun):
        gpu.rope_rows(x, 0, 256, pos[:3], None, 4, 4, 64, 64, THETA)
    with pytest.raises(InvalidArgument):
        gpu.rope_rows(x, -4, 256, pos, None, 4, 4, 64, 64, THETA)
    with pytest.raises(SliceOverrun):
        gpu.t16_rope_store(x, 0, x, 0, x, 0, 256, pos, pos[:3], pos, None, 4, 4, 64, THETA, 1.0, False,
                           TiledCache16(1, 64, 32))


@pytest.mark.parametrize("offset", [0, 5])
def test_more_rows_than_workgroups(gpu, offset):
    """Rows behind the last workgroup's follow at the launch's stride, alone and with a store."""
    from ttsxabe_amd.gpu import TiledCache16
    rows, hd = 70001, 64
    x = rows_of(7, rows, 3 * hd)
    want = ref.rotate(x.view(rows, 3, hd)[:, :2], torch.arange(rows), hd, THETA)
    tol = allowed(x.view(rows, 3, hd)[:, :2], hd, False, 1.0, False)
    half = allowed(x.view(rows, 3, hd)[:, :2], hd, False, 1.0, True)
    cache = TiledCache16(1, hd, rows + offset, zero=False)
    d, q = x.cuda().view(-1), torch.empty(rows * hd, dtype=torch.float32, device="cuda")
    at = torch.arange(rows, dtype=torch.int32).cuda()
    gpu.t16_rope_store(d, 0, d, hd, d, 2 * hd, 3 * hd, at, torch.zeros_like(at), at + offset, None, rows, 1, hd, THETA, 1.0,
                       False, cache, q_out=q)
    assert ((q.cpu().double().view(rows, hd) - want[:, 0]).abs() <= tol[:, 0]).all()
    k, v = ref.untile(cache.data.cpu(), 1, 1, hd, rows + offset)
    assert ((k[0, 0, offset:].double() - want[:, 1]).abs() <= half[:, 1]).all()
    assert torch.equal(v[0, 0, offset:], x[:, 2 * hd:].half())
    gpu.rope_rows(d, 0, 3 * hd, 0, None, rows, 2, hd, hd, THETA)
    got = d.cpu().view(rows, 3, hd)
    assert ((got[:, :2].double() - want).abs() <= tol).all()
    assert torch.equal(got[:, 2], x[:, 2 * hd:])
