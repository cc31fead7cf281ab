"""Queries rotated in place lie over no row of the keys and values that the same
launch reads: refused before any launch, on a machine with no GPU."""
import pytest
import torch

from test_ranges_abi import X, store

STACKED = dict(q_out=X, q_out_stride=6144)  # 32 heads of q, then 8 of k and 8 of v, of 128 dims: rows of 6144


@pytest.mark.parametrize("where", [
    dict(k_off=4095), dict(k_off=0), dict(v_off=4000), dict(v_off=0), dict(q_off=1, k_off=4096),
    dict(q_off=2048, k_off=0, v_off=1025), dict(k_off=4095 + 2 * 6144), dict(k_off=5121, v_off=4096),  # past a row's end
    dict(k_stride=7168), dict(rows=1, k_off=4095), dict(heads=40, q_stride=8192, q_out_stride=8192),
], ids=str)
def test_queries_in_place_over_keys_or_values(where):
    assert store(**{**STACKED, **where}) == 10


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 9, 70])
@pytest.mark.parametrize("order", ["qkv", "kvq", "kqv", "apart"])
def test_queries_in_place_beside_keys_and_values(gpu, rows, order):
    import ranges_ref as ref
    from test_rotary_gpu import THETA, allowed
    from ttsxabe_amd.gpu import TiledCache16
    heads, kv, hd, cap = 4, 2, 64, 96
    part = {"q": heads * hd, "k": kv * hd, "v": kv * hd}
    g = torch.Generator().manual_seed(rows)
    if order == "apart":
        width, off = heads * hd, dict(q=0, k=0, v=0)
        x = {p: torch.randn(rows * width, generator=g) for p in part}
        d = {p: x[p].cuda() for p in part}
    else:
        width, off, at = sum(part.values()), {}, 0
        for p in order:
            off[p], at = at, at + part[p]
        one = torch.randn(rows * width, generator=g)
        x, d = dict.fromkeys(part, one), dict.fromkeys(part, one.cuda())
    row = torch.arange(rows, dtype=torch.int32, device="cuda")
    cache = TiledCache16(kv, hd, cap)
    gpu.t16_rope_store(d["q"], off["q"], d["k"], off["k"], d["v"], off["v"], width, row, torch.zeros_like(row), row, None,
                       rows, heads, hd, THETA, 1.0, False, cache)
    h = {p: x[p].view(rows, width)[:, off[p]:off[p] + part[p]].reshape(rows, -1, hd) for p in part}
    got = d["q"].cpu().view(rows, width)[:, off["q"]:off["q"] + part["q"]].reshape(rows, -1, hd).double()
    assert ((got - ref.rotate(h["q"], row.cpu(), hd, THETA)).abs() <= allowed(h["q"], hd, False, 1.0, False)).all()
    k1, v1 = ref.untile(cache.data.cpu(), 1, kv, hd, cap)
    tol = allowed(h["k"], hd, False, 1.0, True)
    assert ((k1[0, :, :rows].transpose(0, 1).double() - ref.rotate(h["k"], row.cpu(), hd, THETA)).abs() <= tol).all()
    assert torch.equal(v1[0, :, :rows].transpose(0, 1), h["v"].half())
    assert torch.equal(d["k"].cpu().view(rows, width)[:, off["k"]:off["k"] + part["k"]].reshape(rows, -1, hd), h["k"])
