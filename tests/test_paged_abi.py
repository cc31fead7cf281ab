"""Refusals of the paged cache's entry points: argument checks that come before
any launch, so that they run without a GPU."""
import ctypes as C

import pytest

from test_abi import NULL, last
from ttsxabe_amd import _lib

F = C.c_float
BIG = 10**9
P = 16  # a pointer that no refused call follows


def store(**c):
    a = dict(q=P, q_len=BIG, q_off=0, q_stride=4096, q_out=1 << 40, q_out_len=BIG, q_out_off=0, q_out_stride=4096, f16=0,
             k=1 << 41, k_len=BIG, k_off=0, k_stride=4096, v=1 << 42, v_len=BIG, v_off=0, v_stride=4096, pos=P, seq=P,
             index=P, index_len=BIG, table=P, table_len=BIG, table_rows=4, table_cols=16, div=NULL, div_len=0, rows=3,
             heads=8, kv=2, hd=128, rot=128, theta=F(1e4), mscale=F(1.0), inter=0, cache=1 << 43, cache_len=BIG, pages=8,
             page=64)
    a.update(c)
    return _lib.lib().llmtie_paged_rope_store(NULL, *a.values())


def plan(**c):
    a = dict(tk=P, row=NULL, lo=NULL, nseq=3, starts=P, prefix=P, groups=1, max_tk=1000, window=0, shared=0, table_rows=4,
             table_cols=16, page=64, heads=8, kv=2, hd=128, plan=P, plan_len=BIG)
    a.update(c)
    return _lib.lib().llmtie_page_plan(NULL, *a.values())


def attn(**c):
    a = dict(q=P, q_len=BIG, q_off=0, q_stride=1024, cache=P, cache_len=BIG, pages=8, page=64, table=P, table_len=BIG,
             table_rows=4, table_cols=16, tk=P, plan=P, plan_len=BIG, nseq=3, groups=1, max_tk=1000, heads=8, kv=2, hd=128,
             scale=F(0.1), softcap=F(0.0), slopes=NULL, slopes_len=0, ws=P, ws_len=BIG, out=P, out_len=BIG)
    a.update(c)
    return _lib.lib().llmtie_attn_decode_paged(NULL, *a.values())


def selected(**c):
    a = dict(q=P, q_len=BIG, q_off=0, q_stride=1024, cache=P, cache_len=BIG, pages=8, page=64, table=P, table_len=BIG,
             table_rows=4, table_cols=16, tk=P, row=NULL, chosen=P, chosen_len=BIG, count=5, nseq=3, heads=8, kv=2, hd=128,
             scale=F(0.1), softcap=F(0.0), slopes=NULL, slopes_len=0, ws=P, ws_len=BIG, out=P, out_len=BIG)
    a.update(c)
    return _lib.lib().llmtie_attn_decode_selected(NULL, *a.values())


def bounds(**c):
    a = dict(cache=P, cache_len=BIG, pages=8, page=64, table=P, table_len=BIG, table_rows=4, table_cols=16, row=NULL,
             low=NULL, tk=P, nseq=3, max_new=1, kv=2, hd=128, bounds=P, bounds_len=BIG)
    a.update(c)
    return _lib.lib().llmtie_page_bounds(NULL, *a.values())


def select(**c):
    a = dict(q=P, q_len=BIG, q_off=0, q_stride=1024, bounds=P, bounds_len=BIG, pages=8, page=64, table=P, table_len=BIG,
             table_rows=4, table_cols=16, tk=P, row=NULL, nseq=3, max_tk=1000, heads=8, kv=2, hd=128, count=5, first=1,
             last=1, ws=P, ws_len=BIG, chosen=P, chosen_len=BIG)
    a.update(c)
    return _lib.lib().llmtie_select_pages(NULL, *a.values())


ALL = [store, plan, attn, selected, bounds, select]


@pytest.mark.parametrize("call", ALL)
def test_pages_and_tables(call):
    for page in (0, 16, 48, 8192, 2**40):
        assert call(page=page) in (3, 4, 10), page
    assert call(page=33) == 10 and b"power of two" in last().message
    assert call(table_cols=2**25) == 4  # 2^31 positions
    assert call(table_rows=2**31) == 4
    if call is not plan:
        assert call(table_rows=2**30, table_cols=2) == 4 and list(last().field)[:2] == [2**31, BIG]
        assert call(table=NULL) == 10 or call is store
        assert call(pages=2**31) == 4
    if call not in (plan, select):
        need = 8 * _lib.lib().llmtie_t16_cache_len(2, 128, 64)
        assert call(cache_len=need - 1) == 4 and list(last().field)[:2] == [need, need - 1]
        assert call(cache=8) == 10 or call is store


@pytest.mark.parametrize("call", [plan, attn, selected, select])
def test_heads(call):
    for bad in (dict(hd=96), dict(heads=9), dict(kv=0), dict(heads=34, kv=2), dict(heads=0)):
        assert call(**bad) == 1, bad


@pytest.mark.parametrize("call", [plan, selected, bounds, select])
def test_rows_without_a_row_array(call):
    assert call(nseq=5) == 4 and list(last().field)[:2] == [5, 4]


@pytest.mark.parametrize("call", [plan, attn, select])
def test_lengths(call):
    assert call(max_tk=0) == 3 and call(max_tk=16 * 64 + 1) == 3
    assert list(last().field)[:2] == [1025, 1024]


@pytest.mark.parametrize("call", [attn, selected])
def test_attention(call):
    assert call(q_len=1023) == 4 and call(q_stride=1023) == 4 and call(out_len=3 * 1024 - 1) == 4
    assert call(q_off=2**64 - 1) == 4
    for s in (0.0, -1.0, 1e16, float("nan"), float("inf")):
        assert call(scale=F(s)) == 10
    for s in (-1.0, 1e-4, 1e4, float("nan")):
        assert call(softcap=F(s)) == 10
    assert call(slopes=P, slopes_len=7) == 4
    assert call(out=8) == 10
    for name in ("q", "tk", "out", "cache", "table"):
        assert call(**{name: NULL}) == 10, name
    assert call(nseq=0) == 0


def test_plan():
    L = _lib.lib()
    need = L.llmtie_page_plan_len(3, 1, 1000, 4, 8, 2)
    assert plan(plan_len=need - 1) == 4 and list(last().field)[:2] == [need, need - 1]
    assert attn(plan_len=need - 1) == 4
    assert plan(groups=1025) == 4 and plan(nseq=2**20 + 1, row=P) == 4
    for name in ("tk", "plan", "starts", "prefix"):
        assert plan(**{name: NULL}) == 10, name
    assert plan(nseq=0) == 0
    assert L.llmtie_page_plan_len(2**64 - 1, 1, 1000, 4, 8, 2) == 0 and L.llmtie_page_plan_len(3, 1, 1000, 4, 9, 2) == 0
    floats = L.llmtie_attn_paged_workspace(3, 1, 1000, 4, 8, 2, 128)
    assert attn(ws_len=floats - 1) == 4 and attn(ws=NULL) == 10 and attn(ws=8) == 10
    # Short rows that share nothing need none.
    assert L.llmtie_attn_paged_workspace(3, 0, 500, 4, 8, 2, 128) == 0


def test_selected():
    L = _lib.lib()
    assert selected(chosen_len=29) == 4 and list(last().field)[:2] == [30, 29]
    assert selected(chosen=NULL) == 10
    assert selected(count=2**30) == 4
    floats = L.llmtie_attn_selected_workspace(3, 5, 64, 4, 8, 2, 128)
    assert floats and selected(ws_len=floats - 1) == 4 and selected(ws=NULL) == 10 and selected(ws=8) == 10


def test_bounds():
    assert bounds(hd=96) == 1 and bounds(kv=0) == 1
    assert bounds(bounds_len=8 * 2 * 2 * 128 - 1) == 4
    assert bounds(bounds=8) == 10 and bounds(tk=NULL) == 10 and bounds(bounds=NULL) == 10
    assert bounds(nseq=2**24, row=P, table_cols=16) == 4
    assert bounds(nseq=0) == 0 and bounds(pages=0, cache_len=0, bounds_len=0) == 0


def test_select():
    L = _lib.lib()
    assert select(count=0) == 10 and select(count=5, first=3, last=3) == 10 and select(first=2**64 - 1) == 10
    assert select(bounds_len=8 * 2 * 2 * 128 - 1) == 4 and select(bounds=8) == 10
    assert select(q_len=1023) == 4 and select(q_stride=1) == 4 and select(chosen_len=29) == 4
    need = L.llmtie_select_pages_workspace(3, 1000, 64, 5, 2)
    assert need >= 3 * 2 * 16 and select(ws_len=need - 1) == 4 and select(ws=NULL) == 10
    assert L.llmtie_select_pages_workspace(3, 1000, 64, 16, 2) == 0  # all are selected
    for name in ("q", "bounds", "tk", "chosen"):
        assert select(**{name: NULL}) == 10, name
    assert select(nseq=0) == 0


def test_store():
    assert store(table=NULL) == 10
    assert store(index_len=2) == 4 and store(q_stride=1) == 4 and store(k_len=10) == 4
    assert store(rot=127) == 7 and store(hd=96) == 1
    assert store(rows=0) == 0
    assert store(q_out=1 << 41) == 10  # over k's rows


def test_groups_of_a_step():
    """Which sequences a step of LlamaPages attends together, and no more groups of them than a plan takes."""
    from ttsxabe_amd.stack import LlamaPages
    x = LlamaPages.__new__(LlamaPages)
    x.page, x.own = 32, [[5], [1, 2, 9], [7, 8], [1, 2, 3], [6], [1, 2, 4, 10]]
    order, starts, prefix = x._groups([0, 1, 2, 3, 4, 5])
    assert order == [3, 5, 1, 0, 4, 2] and starts == [0, 3, 6] and prefix == [64, 0]
    x.own = [[2 * t + 10**6, t + 10**7] for t in range(3000)]
    assert x._groups(list(range(3000)))[1:] == ([0, 3000], [0])
    x.own = [[t // 2, t + 10**7] for t in range(3000)]
    order, starts, prefix = x._groups(list(range(3000)))
    assert len(prefix) == 1024 and starts[-2:] == [2046, 3000] and prefix == [32] * 1023 + [0]
