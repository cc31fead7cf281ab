"""The refusals of the entry points over key ranges and of the rotary positions
by row: before any launch, on a machine with no GPU."""
import ctypes as C
import math

import pytest
import torch

from ttsxabe_amd import _lib

F, N, BIG, W = C.c_float, None, 10**9, 2**64
X = 4096  # an address that is never read


def status(name, *args):
    return getattr(_lib.lib(), name)(*args)


def ranges(starts=N, starts_len=0, prefix=N, prefix_len=0, rows=8, past=0, window=0, shared=0, table=X, table_len=24,
           pos=N, pos_len=0):
    return status("llmtie_key_ranges", N, starts, starts_len, prefix, prefix_len, rows, past, 1, window, shared, table,
                  table_len, pos, pos_len)


def test_key_ranges():
    assert ranges(table_len=23) == 4
    assert ranges(table=N) == 10
    assert ranges(pos=X, pos_len=7) == 4
    assert ranges(starts=X, starts_len=0) == 4
    assert ranges(starts=X, starts_len=3, prefix=X, prefix_len=1) == 4
    assert ranges(past=2**31 - 4) == 4
    assert ranges(past=W - 4) == 4
    assert ranges(rows=W // 3 + 1, table_len=BIG) == 4
    assert ranges(rows=0, table=N, table_len=0) == 0


def rope(x=X, x_len=BIG, off=0, stride=512, out=X, out_len=BIG, out_off=0, out_stride=512, f16=0, pos=N, pos_len=0,
         first=0, div=N, div_len=0, t=4, heads=4, hd=128, rot=128, theta=1e4, mscale=1.0):
    return status("llmtie_rope_rows", N, x, x_len, off, stride, out, out_len, out_off, out_stride, f16, pos, pos_len,
                  first, div, div_len, t, heads, hd, rot, F(theta), F(mscale), 0)


def test_rope_rows():
    assert rope(hd=127) == 7
    assert rope(hd=0) == 7
    assert rope(rot=63) == 7
    assert rope(rot=130) == 4
    assert rope(hd=2048, stride=8192, out_stride=8192) == 10
    assert rope(theta=0.0) == 10 and rope(theta=math.nan) == 10 and rope(theta=math.inf) == 10
    assert rope(mscale=math.nan) == 10
    assert rope(x_len=4 * 512 - 1) == 4
    assert rope(out=2**40, out_len=4 * 512 - 1) == 4
    assert rope(stride=511) == 4 and rope(out_stride=511) == 4
    assert rope(off=W - 1) == 4 and rope(out_off=W - 512) == 4 and rope(stride=W // 2) == 4
    assert rope(pos=X, pos_len=3) == 4
    assert rope(div=X, div_len=63) == 4
    assert rope(first=2**31 - 2) == 4
    assert rope(x=N) == 10 and rope(out=N) == 10
    # Over its own rows, or apart from them: no other overlap.
    assert rope(out_off=512) == 10
    assert rope(out_stride=1024) == 10
    assert rope(f16=1) == 10
    assert rope(t=0, x=N, out=N) == 0 and rope(heads=0, x=N, out=N) == 0


def store(q=X, q_len=BIG, q_off=0, q_stride=6144, q_out=2**40, q_out_len=BIG, q_out_off=0, q_out_stride=4096, f16=0,
          k=X, k_len=BIG, k_off=4096, k_stride=6144, v=X, v_len=BIG, v_off=5120, v_stride=6144, pos=X, slot=X, index=X,
          index_len=4, div=N, div_len=0, rows=4, heads=32, kv=8, hd=128, rot=128, cache=2**41, cache_len=BIG, slots=2,
          cap=512):
    return status("llmtie_t16_rope_store", N, q, q_len, q_off, q_stride, q_out, q_out_len, q_out_off, q_out_stride, f16,
                  k, k_len, k_off, k_stride, v, v_len, v_off, v_stride, pos, slot, index, index_len, div, div_len, rows,
                  heads, kv, hd, rot, F(1e4), F(1.0), 0, cache, cache_len, slots, cap)


def test_rope_store():
    assert store(hd=96) == 1 and store(kv=0) == 1
    assert store(index_len=3) == 4
    assert store(cache_len=2 * 8 * 512 * 128 * 2 - 1) == 4
    assert store(cap=2**31) == 4 and store(slots=2**31) == 4
    assert store(q_len=4095) == 4 and store(k_len=5119) == 4 and store(v_len=6143) == 4
    assert store(q_out_len=4 * 4096 - 1) == 4
    assert store(q_stride=4095) == 4 and store(q_out_stride=4095) == 4 and store(k_stride=1023) == 4
    assert store(v_stride=1023) == 4
    assert store(k_off=W - 1) == 4 and store(v_off=W - 1024) == 4
    for hole in ("k", "v", "pos", "slot", "index", "cache", "q_out"):
        assert store(**{hole: N}) == 10, hole
    assert store(cache=2**41 + 8) == 10
    assert store(q_out=X, q_out_stride=4096) == 10  # over the stacked rows, but not its own
    assert store(rot=130) == 4 and store(div=X, div_len=63) == 4
    assert store(rows=0, q=N, k=N, v=N) == 0


def prompt(q=X, q_len=BIG, q_off=0, q_stride=4096, cache=2**41, cache_len=BIG, slots=1, slot=0, table=X, table_len=12,
           out=2**40, out_len=BIG, tq=4, past=0, heads=32, kv=8, hd=128, cap=512, scale=0.1, softcap=0.0, slopes=N,
           slopes_len=0, max_keys=0, ws=N, ws_len=0):
    return status("llmtie_flash_attn_ranges_t16", N, q, q_len, q_off, q_stride, cache, cache_len, slots, slot, table,
                  table_len, max_keys, out, out_len, tq, past, heads, kv, hd, cap, F(scale), F(softcap), slopes,
                  slopes_len, ws, ws_len)


def test_prompts():
    assert prompt(hd=96) == 1 and prompt(kv=5) == 1 and prompt(kv=0) == 1
    assert prompt(past=509) == 3 and prompt(past=W - 2) == 3
    for scale in (0.0, -1.0, math.nan, math.inf):
        assert prompt(scale=scale) == 10
    for cap in (-1.0, 1e-4, 2e3, math.nan, math.inf):
        assert prompt(softcap=cap) == 10
    assert prompt(slopes=X, slopes_len=31) == 4
    assert prompt(slot=1) == 4 and prompt(slots=0) == 4
    assert prompt(cache_len=8 * 512 * 128 * 2 - 1) == 4
    assert prompt(q_stride=4095) == 4 and prompt(q_len=4 * 4096 - 1) == 4 and prompt(q_off=W - 1) == 4
    assert prompt(out_len=4 * 4096 - 1) == 4
    assert prompt(table_len=11) == 4 and prompt(table_len=15) == 10
    for hole in ("q", "cache", "table", "out"):
        assert prompt(**{hole: N}) == 10, hole
    assert prompt(cache=2**41 + 2) == 10 and prompt(out=2**40 + 8) == 10
    assert prompt(cap=2**31 - 1, cache_len=2**62) == 4
    assert prompt(tq=0, q=N, table_len=0) == 0


def test_prompt_workspace():
    size = _lib.lib().llmtie_flash_attn_ranges_workspace
    assert size(0, 4096, 32, 8, 128) == 0
    assert size(16, 4096, 32, 8, 96) == 0 and size(16, 4096, 32, 0, 128) == 0
    assert size(16, 300, 32, 8, 128) == 0  # too few keys to cut
    assert size(8192, 8192, 32, 8, 128) == 0  # enough rows
    n = size(16, 4096, 32, 8, 128)
    assert n > 0 and n % (16 * 32 * 130) == 0
    assert prompt(tq=16, past=4080, cap=4096, table_len=48, ws=2**42, ws_len=n - 1) == 4
    assert prompt(tq=16, past=4080, cap=4096, table_len=48, ws=2**42 + 4, ws_len=n) == 10


def decode(q=X, q_len=BIG, q_off=0, q_stride=4096, cache=2**41, cache_len=BIG, slots=3, tk=X, slot=X, nseq=3,
           max_tk=512, window=0, shared=0, heads=32, kv=8, hd=128, cap=512, scale=0.1, softcap=0.0, slopes=N,
           slopes_len=0, out=2**40, out_len=BIG, scratch=N):
    return status("llmtie_attn_decode_ranges_t16", N, q, q_len, q_off, q_stride, cache, cache_len, slots, tk, slot, N,
                  nseq, max_tk, window, shared, heads, kv, hd, cap, F(scale), F(softcap), slopes, slopes_len, scratch,
                  out, out_len)


def test_decode():
    assert decode(hd=96) == 1 and decode(kv=5) == 1 and decode(heads=34, kv=2) == 1
    assert decode(max_tk=513) == 3 and decode(max_tk=0) == 3
    assert decode(scale=-1.0) == 10 and decode(softcap=-1.0) == 10 and decode(scale=math.nan) == 10
    assert decode(slopes=X, slopes_len=31) == 4
    assert decode(cache_len=3 * 8 * 512 * 128 * 2 - 1) == 4
    assert decode(q_stride=4095) == 4 and decode(q_len=3 * 4096 - 1) == 4 and decode(q_off=W - 1) == 4
    assert decode(out_len=3 * 4096 - 1) == 4
    assert decode(slot=N, slots=2) == 4
    for hole in ("q", "cache", "tk", "out", "scratch"):
        assert decode(**{hole: N}) == 10, hole
    assert decode(nseq=0, q=N) == 0
    s = _lib.lib().llmtie_decode_scratch_new()
    try:
        assert decode(scratch=s, cache=2**41 + 4) == 10 and decode(scratch=s, out=2**40 + 4) == 10
        # More workgroups than a launch holds.
        assert decode(scratch=s, nseq=2**22, cache_len=2**62, slots=2**22, q_len=2**62, out_len=2**62) == 4
    finally:
        _lib.lib().llmtie_decode_scratch_free(s)


def test_scaling_tables():
    from ttsxabe_amd.gpu import InvalidArgument, OddHeadDim, rope_scaling
    assert rope_scaling(128, 500000.0, device="cpu") == (None, 500000.0, 1.0)
    d, t, m = rope_scaling(64, 1e4, "linear", 4.0, device="cpu")
    assert t == 1e4 and m == 1.0 and torch.equal(d, torch.full((32,), 4.0))
    d, t, m = rope_scaling(64, 1e4, "ntk", 4.0, device="cpu")
    assert d is None and m == 1.0
    assert math.isclose(t ** (-62 / 64), 1e4 ** (-62 / 64) / 4.0, rel_tol=1e-12)  # the slowest frequency
    d, t, m = rope_scaling(128, 1e4, "yarn", 8.0, original=4096, device="cpu")
    assert t == 1e4 and math.isclose(m, 1.0 + 0.1 * math.log(8.0))
    turns = 4096 / (2 * math.pi) * 1e4 ** (-torch.arange(64, dtype=torch.float64) / 64)
    assert (d[turns > 34.0] == 1.0).all() and (d[turns < 0.85] == 8.0).all()
    assert (d[1:] >= d[:-1]).all() and ((d > 1.0) & (d < 8.0)).any()
    with pytest.raises(InvalidArgument):
        rope_scaling(64, 1e4, "other")
    with pytest.raises(InvalidArgument):
        rope_scaling(64, 1e4, "yarn", 0.5)
    with pytest.raises(OddHeadDim):
        rope_scaling(63, 1e4, "linear", 2.0)


def test_rotary_sizes():
    """A row index behind the last workgroup's stays an int, and so do a thread's items."""
    n = 2**26
    assert rope(t=n + 1, heads=1, hd=2, rot=2, stride=2, out_stride=2) == 4
    assert rope(t=2**31 - 1, heads=1, hd=2, rot=2, stride=2, out_stride=2) == 4
    assert rope(t=1, heads=2**22 + 1, stride=2**29 + 128, out_stride=2**29 + 128) == 4
    assert store(rows=n + 1, index_len=n + 1) == 4
    assert store(q=N, rows=1, kv=2**23 + 1, hd=64, rot=64, k_stride=2**30, v_stride=2**30, slots=1, cap=32,
                 cache_len=2**62) == 4


def test_score_scales():
    for scale in (9e-16, 1.1e15, 1e30, 1e-30):
        assert prompt(scale=scale) == 10 and decode(scale=scale) == 10, scale


def test_scaling_refusals():
    from ttsxabe_amd.gpu import InvalidArgument, rope_scaling
    for theta in (1.0, 0.5, math.nan):
        with pytest.raises(InvalidArgument):
            rope_scaling(64, theta, "yarn", 4.0, device="cpu")
    for kind in ("linear", "ntk", "yarn"):
        for factor in (math.inf, math.nan, 0.0):
            with pytest.raises(InvalidArgument):
                rope_scaling(64, 1e4, kind, factor, device="cpu")


def test_a_gguf_that_rotates_a_part_of_its_heads(tmp_path):
    """Its own order keeps the count of rotated dims; unpermuted (whole) heads are rotated whole, as before."""
    import numpy as np

    from oracle.stack import StackConfig, random_weights
    from tests.test_gguf import llama_gguf
    from ttsxabe_amd.llama_gguf import load_llama_gguf
    cfg = StackConfig()
    llama_gguf(tmp_path / "m.gguf", cfg, random_weights(cfg, 1))
    f = load_llama_gguf(tmp_path / "m.gguf")[0]
    assert f.rope_dim == 0 and not f.rope_interleaved
    from ttsxabe_amd import llama_gguf as m
    config = m.config_from_gguf
    try:
        m.config_from_gguf = lambda f: m.replace(config(f), rope_dim=cfg.head_dim // 2)
        whole, a = m.load_llama_gguf(tmp_path / "m.gguf")
        part, b = m.load_llama_gguf(tmp_path / "m.gguf", interleaved=True)
    finally:
        m.config_from_gguf = config
    assert whole.rope_dim == 0 and part.rope_dim == cfg.head_dim // 2 and part.rope_interleaved
    assert np.array_equal(m.unpermute_rope(b["0.wq"], cfg.heads), a["0.wq"])


@pytest.mark.parametrize("names", ["Gpu, DecodeScratch, TiledCache16, KeyRanges, rope_scaling", "gpu", "rope_scaling"])
def test_names_of_the_package(names):
    """In a process that has not imported the mirror yet."""
    import subprocess
    import sys
    from pathlib import Path
    subprocess.run([sys.executable, "-c", f"from ttsxabe_amd import {names}"], check=True,
                   cwd=Path(__file__).resolve().parent.parent)
