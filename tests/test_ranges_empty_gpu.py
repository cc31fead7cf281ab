"""Arrays that are given but too short for the call, down to empty ones, are
refused: they are not taken for arrays that are not given."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def floats(n):
    return torch.ones(n, device="cuda")


def test_row_tables(gpu):
    from ttsxabe_amd.gpu import SliceOverrun
    for short in (dict(starts=ints()), dict(prefix=ints()), dict(starts=ints(0, 3, 7), prefix=ints(1)),
                  dict(starts=ints(0, 3, 7), prefix=ints())):
        with pytest.raises(SliceOverrun):
            gpu.key_ranges(7, **short)
    r = gpu.key_ranges(7, starts=ints(2), prefix=ints())  # no documents, none of which has a prefix
    assert not r.table.any() and not r.pos.any()


@pytest.mark.parametrize("n", [0, 1, 31])
def test_rotations(gpu, n):
    from ttsxabe_amd.gpu import SliceOverrun, TiledCache16
    heads, hd, rows = 2, 64, 32
    x = torch.randn(rows * 3 * heads * hd, device="cuda")
    before = x.clone()
    with pytest.raises(SliceOverrun):
        gpu.rope_rows(x, 0, heads * hd, 0, floats(n), rows, heads, hd, hd, 1e4)
    with pytest.raises(SliceOverrun):
        gpu.rope_rows(x, 0, heads * hd, ints(*range(n)), None, rows, heads, hd, hd, 1e4)
    cache = TiledCache16(heads, hd, 64)
    full = ints(*range(rows)), torch.zeros(rows, dtype=torch.int32, device="cuda"), ints(*range(rows))

    def store(pos, slot, index, div):
        gpu.t16_rope_store(None, 0, x, 0, x, heads * hd, 3 * heads * hd, pos, slot, index, div, rows, heads, hd, 1e4, 1.0,
                           False, cache)
    for i in range(3):
        with pytest.raises(SliceOverrun):
            store(*(t[:n] if i == j else t for j, t in enumerate(full)), None)
    with pytest.raises(SliceOverrun):
        store(*full, floats(n))
    assert torch.equal(x, before) and not cache.data.any()
    gpu.rope_rows(x, 0, heads * hd, ints(), floats(0), 0, heads, hd, 0, 1e4)  # no rows, no dims: none needed
    assert torch.equal(x, before)


@pytest.mark.parametrize("n", [0, 3])
def test_attention(gpu, n):
    from ttsxabe_amd.gpu import DecodeScratch, SliceOverrun, TiledCache16
    heads, hd, rows = 4, 64, 5
    cache = TiledCache16(2, hd, 32, slots=rows)
    q = torch.randn(rows * heads * hd, device="cuda")
    with pytest.raises(SliceOverrun):
        gpu.flash_attn_ranges(q.half(), 0, heads * hd, cache, 0, gpu.key_ranges(rows), rows, 0, heads, 0.1, 0.0, floats(n))
    lens, s = ints(1, 2, 3, 4, 5), DecodeScratch()
    for short in (dict(slopes=floats(n)), dict(lo_dev=lens[:n])):
        with pytest.raises(SliceOverrun):
            gpu.attn_decode_ranges(q, 0, heads * hd, cache, lens, None, 32, heads, 0.1, s, **short)
    with pytest.raises(SliceOverrun):
        gpu.attn_decode_ranges(q, 0, heads * hd, cache, lens, lens[:n], 32, heads, 0.1, s)
