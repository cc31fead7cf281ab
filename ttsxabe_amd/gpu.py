"""Host-side mirror of the reference's attention operators, over the C ABI.

`Gpu` has the methods of `llmtie_cuda::Gpu` that the attention path uses
(crates/llmtie-cuda/src/device.rs:2849-3190, :5410-5470, :5697-6410), with the
same names, argument order and meaning; device slices are torch tensors on
the GPU (torch is only the allocator and the stream here). Outputs are
allocated by the callee exactly where the reference allocates them. Errors are
raised as the reference's `CudaError` variants (error.rs:148-282), before any
launch, from the library's own checks.

There is no CPU fallback: constructing a `Gpu` without the built library or
without a HIP device raises.
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass

import torch

from . import _lib

__all__ = [
    "CudaError", "UnsupportedAttention", "OddCacheCapacity", "CacheOverrun", "SliceOverrun", "RaggedBlock",
    "MismatchedQ8", "OddHeadDim", "Driver", "NoDevice", "InvalidArgument", "ScratchGrowthInCapture", "ScratchLimit",
    "SplitHeadLost",
    "DecodeScratch",
    "Q8", "KvCacheQ8",
    "TiledCache16", "KeyRanges", "rope_scaling", "PagedCache16", "PagePlan", "Gpu",
]


class CudaError(RuntimeError):
    """Base of the named refusals (error.rs)."""

    status = -1

    def __init__(self, message: str, fields=()):
        super().__init__(message)
        self.fields = tuple(fields)


class UnsupportedAttention(CudaError):
    status = 1


class OddCacheCapacity(CudaError):
    status = 2


class CacheOverrun(CudaError):
    status = 3


class SliceOverrun(CudaError):
    status = 4


class RaggedBlock(CudaError):
    status = 5


class MismatchedQ8(CudaError):
    status = 6


class OddHeadDim(CudaError):
    status = 7


class Driver(CudaError):
    status = 8


class NoDevice(CudaError):
    status = 9


class InvalidArgument(CudaError):
    status = 10


class ScratchGrowthInCapture(CudaError):
    """A decode scratch would have to grow while its stream captures a graph."""
    status = 11


class ScratchLimit(CudaError):
    """The fixed scratch of attn_decode_f16_noalloc is too small for the call."""
    status = 12


class SplitHeadLost(CudaError):
    """An earlier decode through this scratch wrote NaN for a head whose split
    workgroups did not share an XCD (the XCD-local hand-off's self-check)."""
    status = 13


_BY_STATUS = {c.status: c for c in (UnsupportedAttention, OddCacheCapacity, CacheOverrun, SliceOverrun,
                                    RaggedBlock, MismatchedQ8, OddHeadDim, Driver, NoDevice, InvalidArgument,
                                    ScratchGrowthInCapture, ScratchLimit, SplitHeadLost)}


def _check(status: int):
    if status == 0:
        return
    err = _lib.LlmtieError()
    _lib.lib().llmtie_last_error(C.byref(err))
    cls = _BY_STATUS.get(status, CudaError)
    raise cls(err.message.decode(errors="replace"), [err.field[i] for i in range(4)])


def _p(t):
    """Device pointer of a tensor (None -> NULL), as the plain integer the
    declared argument types take."""
    return None if t is None else t.data_ptr()


def _n(t):
    return 0 if t is None else t.numel()


def _need(t, dtypes, what):
    if t is None or (t.is_cuda and t.dtype in dtypes and t.is_contiguous()):
        return
    if not t.is_cuda:
        raise InvalidArgument(f"{what} is not a device tensor")
    if t.dtype not in dtypes:
        raise InvalidArgument(f"{what} has dtype {t.dtype}, wanted one of {dtypes}")
    raise InvalidArgument(f"{what} is not contiguous")


_F32 = (torch.float32,)
_H16 = (torch.float16, torch.int16, torch.uint16) if hasattr(torch, "uint16") else (torch.float16, torch.int16)
_I8 = (torch.int8,)
_I32 = (torch.int32,)


class DecodeScratch:
    """What the decode keeps between calls (device.rs:208-231): split partials
    and arrival counters, caller-owned, grown on demand."""

    def __init__(self):
        self._h = _lib.lib().llmtie_decode_scratch_new()
        if not self._h:
            raise Driver("could not allocate a decode scratch")

    @property
    def handle(self):
        return self._h

    def check(self):
        """Raises SplitHeadLost if an earlier decode through this scratch lost
        a head to the XCD-local check (read after a synchronisation); the
        status is cleared."""
        _check(_lib.lib().llmtie_decode_scratch_status(self._h))

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h:
            try:
                _lib.lib().llmtie_decode_scratch_free(h)
            except Exception:
                pass


@dataclass
class Q8:
    """An int8 twin: `rows * k` codes then `rows * k / 32` f32 scales in one
    buffer (device.rs:498-520)."""

    buf: torch.Tensor
    rows: int
    k: int

    def scale_offset(self) -> int:
        return self.rows * self.k

    def shape(self):
        return (self.rows, self.k)

    def parts(self):
        """(codes int8 [rows*k], scales f32 [rows*k/32]) on the host."""
        raw = self.buf.cpu()
        codes = raw[: self.scale_offset()].clone()
        scales = raw[self.scale_offset(): self.scale_offset() + self.rows * self.k // 32 * 4].view(torch.float32)
        return codes, scales.clone()


class KvCacheQ8:
    """A tiled GGUF Q8_0 KV cache for `slots` sequences (layout in
    llmtie_hip.h / csrc/kvlayout.h): one int8 buffer of whole 32-position
    blocks, codes and f16 scales of K and V per block."""

    def __init__(self, slots: int, kv_heads: int, head_dim: int, cap: int, device="cuda"):
        self.slots, self.kv_heads, self.head_dim, self.cap = slots, kv_heads, head_dim, cap
        n = _lib.lib().llmtie_q8_cache_bytes(slots, kv_heads, head_dim, cap)
        self.data = torch.zeros(n, dtype=torch.int8, device=device)
        # An empty cache holds code 0 (offset-binary 0x80) with scale 0.
        blocks = self.data.view(-1, n // (slots * kv_heads * ((cap + 31) // 32)))
        blocks[:, : 64 * head_dim].fill_(-128)

    def bytes_per_position(self) -> int:
        """HBM bytes one live position of one sequence costs a decode step."""
        return 2 * self.kv_heads * (self.head_dim + 2 * self.head_dim // 32)


class TiledCache16:
    """A tiled f16 KV cache for one layer: K and V of every kv head in one
    buffer, 32-position blocks in MFMA fragment order; `slots` sequences' one
    after the other (the operators without slots take the first)."""

    def __init__(self, kv_heads: int, head_dim: int, cap: int, device="cuda", zero=True, slots: int = 1):
        self.kv_heads, self.head_dim, self.cap, self.slots = kv_heads, head_dim, cap, slots
        n = slots * _lib.lib().llmtie_t16_cache_len(kv_heads, head_dim, cap)
        alloc = torch.zeros if zero else torch.empty
        self.data = alloc(n, dtype=torch.float16, device=device)

    @classmethod
    def of(cls, data, kv_heads: int, head_dim: int, cap: int, slots: int = 1):
        """A cache over memory that the caller holds."""
        self = cls.__new__(cls)
        self.kv_heads, self.head_dim, self.cap, self.slots, self.data = kv_heads, head_dim, cap, slots, data
        return self


@dataclass
class KeyRanges:
    """Which keys each row of a prompt sees: `table` int32 [3, rows] (row r sees
    keys j < table[0, r] and table[1, r] <= j < table[2, r]), `pos` int32 [rows]
    its rotary positions, `max_keys` a bound of the keys a row sees (0: unknown)."""

    table: torch.Tensor
    pos: torch.Tensor | None = None
    max_keys: int = 0


class PagedCache16(TiledCache16):
    """A tiled f16 cache for one layer in `pages` pages of `page` positions (a
    power of two from 32 to 4096), which are its slots. A sequence's positions lie
    where a row of a table (int32 [rows, pages of the longest]) says."""

    def __init__(self, kv_heads: int, head_dim: int, pages: int, page: int, device="cuda", zero=True):
        super().__init__(kv_heads, head_dim, page, device=device, zero=zero, slots=pages)
        self.pages, self.page = pages, page

    @classmethod
    def of(cls, data, kv_heads: int, head_dim: int, pages: int, page: int):
        """A cache over memory that the caller holds."""
        self = super().of(data, kv_heads, head_dim, page, slots=pages)
        self.pages, self.page = pages, page
        return self


@dataclass
class PagePlan:
    """What Gpu.page_plan made of a step's rows, for the attention of all layers: the
    rows' lengths and tables, which it holds on to, and how the work is divided."""

    data: torch.Tensor
    tk: torch.Tensor
    table: torch.Tensor
    heads: int
    kv_heads: int
    head_dim: int
    page: int
    groups: int
    max_tk: int
    floats: int  # of the attention's workspace


def rope_scaling(rot_dim: int, theta: float, kind: str = "none", factor: float = 1.0, original: int = 8192,
                 beta_fast: float = 32.0, beta_slow: float = 1.0, device="cuda"):
    """(freq_div, theta, mscale) of a rotary extended to `factor` times its
    `original` positions, for rope_rows and t16_rope_store.

    linear: every frequency is divided by the factor. ntk: the base grows to
    theta * factor^(rot / (rot - 2)), which divides the slowest frequency by the
    factor and leaves the fastest. yarn: frequencies that turn more than
    beta_fast times within `original` positions stay, those that turn less than
    beta_slow times are divided by the factor, a ramp over the dims between
    blends the two, and the rotated values are multiplied by 1 + ln(factor) / 10."""
    if kind not in ("none", "linear", "ntk", "yarn"):
        raise InvalidArgument(f"unknown rotary scaling {kind!r}")
    if rot_dim % 2 or rot_dim < 0:
        raise OddHeadDim(f"a rotary head of odd width {rot_dim}", (rot_dim,))
    if not (math.inf > factor >= 1.0 and math.inf > theta > 0.0 and original > 0 and beta_fast > beta_slow > 0.0):
        raise InvalidArgument("a rotary scaling wants factor >= 1, theta, original > 0 and beta_fast > beta_slow > 0")
    n = rot_dim // 2
    if kind == "none" or factor == 1.0 or n == 0:
        return None, theta, 1.0
    if kind == "ntk":
        return None, theta * factor ** (rot_dim / (rot_dim - 2)) if rot_dim > 2 else theta, 1.0
    if kind == "linear":
        return torch.full((n,), factor, dtype=torch.float32, device=device), theta, 1.0
    if not theta > 1.0:
        raise InvalidArgument("yarn wants frequencies that fall: theta > 1")
    # The dim whose frequency turns b times within `original` positions.
    def at(b):
        return n * math.log(original / (b * 2.0 * math.pi)) / math.log(theta)
    first = max(math.floor(at(beta_fast)), 0)
    last = min(math.ceil(at(beta_slow)), rot_dim - 1)
    i = torch.arange(n, dtype=torch.float64)
    ramp = ((i - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)  # 0: kept, 1: divided
    div = 1.0 / ((1.0 - ramp) + ramp / factor)
    return div.to(device=device, dtype=torch.float32), theta, 1.0 + 0.1 * math.log(factor)


class Gpu:
    """The attention operators of `llmtie_cuda::Gpu`, on gfx950."""

    def __init__(self, device: int = 0):
        L = _lib.lib()  # raises if the library is not built
        if not torch.cuda.is_available():
            raise NoDevice("no usable HIP device")
        self.device = torch.device("cuda", device)
        self._L = L

    def _stream(self):
        # The current stream's handle without a Stream object: a call of a few
        # launches is as long as its host work (three calls of the f32 prompt
        # layer took 25.2 us of it with the ctypes and Stream objects, 17.2 us
        # without).
        return torch._C._cuda_getCurrentRawStream(self.device.index)

    # ------------------------------------------------------------- prefill

    def supports_flash(self, head_dim: int, heads: int, kv_heads: int) -> bool:
        return bool(self._L.llmtie_supports_flash(head_dim, heads, kv_heads))

    def _flash(self, fn, q, k, v, tq, past, heads, kv_heads, head_dim, cap, scale, causal, kdt, *ws, split=False):
        _need(q, _F32, "q")
        _need(k, kdt, "k")
        _need(v, kdt, "v")
        out = torch.empty(max(tq * heads * head_dim, 1), dtype=torch.float32, device=self.device)
        # After the output: a card with room for that alone still has its call.
        if split:
            w = self._flash_ws(tq, past, heads, kv_heads, head_dim)
            ws = _p(w), _n(w)
        _check(fn(self._stream(), _p(q), _n(q), _p(k), _n(k), _p(v), _n(v), _p(out), tq * heads * head_dim, tq, past,
                  heads, kv_heads, head_dim, cap, scale, int(bool(causal)), *ws))
        return out[: tq * heads * head_dim]

    def _flash_ws(self, tq, past, heads, kv_heads, head_dim):
        """The workspace of a prefill off an f16 cache (None: it needs none). It
        is a torch allocation of the current stream like the output, so the
        allocator keeps its memory from other streams until the launches on
        this one are done."""
        if past + tq <= 512 or min(tq, past, heads, kv_heads, head_dim) < 0:
            return None  # too few keys to split, or refused by the call itself
        n = self._L.llmtie_flash_attn_workspace(tq, past, heads, kv_heads, head_dim)
        if not n:
            return None
        try:
            return torch.empty(n, dtype=torch.float32, device=self.device)
        except torch.OutOfMemoryError:
            return None  # the unsplit prefill needs nothing beside its output

    def flash_attn(self, q, k, v, tq, past, heads, kv_heads, head_dim, cap, scale, causal):
        """device.rs:5702."""
        return self._flash(self._L.llmtie_flash_attn, q, k, v, tq, past, heads, kv_heads, head_dim, cap, scale,
                           causal, _F32)

    def flash_attn_f16(self, q, k, v, tq, past, heads, kv_heads, head_dim, cap, scale, causal):
        """device.rs:5754. k, v: f16 caches (float16 or 16-bit integer bits)."""
        return self._flash(self._L.llmtie_flash_attn_f16_ws, q, k, v, tq, past, heads, kv_heads, head_dim, cap, scale,
                           causal, _H16, split=True)

    def flash_attn_rows(self, qkv, t, heads, head_dim, scale):
        """device.rs:5812. Returns the f16 context [t * heads * head_dim]."""
        _need(qkv, _F32, "qkv")
        n = t * heads * head_dim
        out = torch.empty(max(n, 1), dtype=torch.float16, device=self.device)
        _check(self._L.llmtie_flash_attn_rows(self._stream(), _p(qkv), _n(qkv), _p(out), n, t, heads, head_dim,
                                              scale))
        return out[:n]

    # -------------------------------------------------------------- decode

    def attn_decode_f16(self, q, k, v, heads, kv_heads, head_dim, tk, cap, scale, scale_q, scratch):
        """device.rs:5949."""
        _need(q, _F32, "q")
        _need(k, _H16, "k")
        _need(v, _H16, "v")
        n = heads * head_dim
        out = torch.empty(n, dtype=torch.float32, device=self.device)
        _check(self._L.llmtie_attn_decode_f16(self._stream(), _p(q), _n(q), _p(k), _n(k), _p(v), _n(v), heads,
                                              kv_heads, head_dim, tk, cap, scale, int(bool(scale_q)),
                                              scratch.handle, _p(out), n))
        return out

    def attn_decode_f16_noalloc(self, q, k, v, heads, kv_heads, head_dim, tk, cap, scale, scale_q, out=None):
        """attn_decode_f16 without a scratch: the library's fixed per-device
        scratch (no reference counterpart; for callers that cannot allocate).
        Calls that can overlap on one device race."""
        _need(q, _F32, "q")
        _need(k, _H16, "k")
        _need(v, _H16, "v")
        _need(out, _F32, "out")
        n = heads * head_dim
        if out is None:
            out = torch.empty(n, dtype=torch.float32, device=self.device)
        _check(self._L.llmtie_attn_decode_f16_noalloc(self._stream(), _p(q), _n(q), _p(k), _n(k), _p(v), _n(v),
                                                      heads, kv_heads, head_dim, tk, cap, scale,
                                                      int(bool(scale_q)), _p(out), _n(out)))
        return out

    def q8_zeros(self, rows: int, k: int) -> Q8:
        """device.rs:1056."""
        if k % 32 != 0:
            raise RaggedBlock(f"a row of {k} in blocks of 32", (k, 32))
        return Q8(torch.zeros(rows * k + rows * (k // 32) * 4, dtype=torch.int8, device=self.device), rows, k)

    def attn_decode_f16_q(self, q, k, v, heads, kv_heads, head_dim, tk, cap, scale, scale_q, scratch):
        """device.rs:5973: the context and its int8 twin."""
        _need(q, _F32, "q")
        _need(k, _H16, "k")
        _need(v, _H16, "v")
        n = heads * head_dim
        out = torch.empty(n, dtype=torch.float32, device=self.device)
        twin = Q8(torch.empty(n + (n // 32) * 4, dtype=torch.int8, device=self.device), 1, n)
        _check(self._L.llmtie_attn_decode_f16_q(self._stream(), _p(q), _n(q), _p(k), _n(k), _p(v), _n(v), heads,
                                                kv_heads, head_dim, tk, cap, scale, int(bool(scale_q)),
                                                scratch.handle, _p(out), n, _p(twin.buf), twin.buf.numel()))
        return out, twin

    def attn_decode_f16_q_row(self, q, q_off, k, v, heads, kv_heads, head_dim, tk, cap, scale, scale_q, scratch,
                              out, twin: Q8, row):
        """device.rs:6001."""
        _need(q, _F32, "q")
        _need(k, _H16, "k")
        _need(v, _H16, "v")
        _need(out, _F32, "out")
        _check(self._L.llmtie_attn_decode_f16_q_row(self._stream(), _p(q), _n(q), q_off, _p(k), _n(k), _p(v), _n(v),
                                                    heads, kv_heads, head_dim, tk, cap, scale,
                                                    int(bool(scale_q)), scratch.handle, _p(out), _n(out),
                                                    _p(twin.buf), twin.rows, twin.k, row))

    def attn_decode(self, q, k, v, heads, kv_heads, head_dim, tk, cap, scale, scale_q, scratch):
        """device.rs:6132: off an f32 cache."""
        _need(q, _F32, "q")
        _need(k, _F32, "k")
        _need(v, _F32, "v")
        n = heads * head_dim
        out = torch.empty(n, dtype=torch.float32, device=self.device)
        _check(self._L.llmtie_attn_decode(self._stream(), _p(q), _n(q), _p(k), _n(k), _p(v), _n(v), heads, kv_heads,
                                          head_dim, tk, cap, scale, int(bool(scale_q)), scratch.handle,
                                          _p(out), n))
        return out

    def attn_decode_q8_batch(self, q, cache: KvCacheQ8, tk_dev, slot_dev, max_tk, heads, scale, scale_q, scratch,
                             out=None):
        """Batched decode of len(tk_dev) sequences over a Q8_0 cache (new)."""
        _need(q, _F32, "q")
        _need(tk_dev, _I32, "tk")
        _need(slot_dev, _I32, "slot")
        nseq = tk_dev.numel()
        n = heads * cache.head_dim
        if out is None:
            out = torch.empty(max(nseq * n, 1), dtype=torch.float32, device=self.device)
        _check(self._L.llmtie_attn_decode_q8_batch(
            self._stream(), _p(q), _n(q), _p(cache.data), _n(cache.data), cache.slots, _p(tk_dev), _p(slot_dev),
            nseq, max_tk, heads, cache.kv_heads, cache.head_dim, cache.cap, scale, int(bool(scale_q)),
            scratch.handle, _p(out), _n(out)))
        return out[: nseq * n]

    # ---------------------------------------------------------- tiled f16

    def attn_decode_t16(self, q, cache: TiledCache16, heads, tk, scale, scale_q, scratch, out=None):
        """attn_decode_f16 (device.rs:5949) off a tiled cache."""
        _need(q, _F32, "q")
        n = heads * cache.head_dim
        if out is None:
            out = torch.empty(n, dtype=torch.float32, device=self.device)
        _check(self._L.llmtie_attn_decode_t16(self._stream(), _p(q), _n(q), _p(cache.data), _n(cache.data), heads,
                                              cache.kv_heads, cache.head_dim, tk, cache.cap, scale,
                                              int(bool(scale_q)), scratch.handle, _p(out), _n(out)))
        return out

    def attn_decode_t16_q_row(self, q, q_off, cache: TiledCache16, heads, tk, scale, scale_q, scratch, out,
                              twin: Q8 = None, row=0):
        """attn_decode_f16_q_row (device.rs:6001) off a tiled cache."""
        _need(q, _F32, "q")
        _need(out, _F32, "out")
        _check(self._L.llmtie_attn_decode_t16_q_row(
            self._stream(), _p(q), _n(q), q_off, _p(cache.data), _n(cache.data), heads, cache.kv_heads,
            cache.head_dim, tk, cache.cap, scale, int(bool(scale_q)), scratch.handle, _p(out), _n(out),
            None if twin is None else _p(twin.buf), 0 if twin is None else twin.rows,
            0 if twin is None else twin.k, row))

    def flash_attn_t16(self, q, cache: TiledCache16, tq, past, heads, scale, causal):
        """flash_attn_f16 (device.rs:5754) off a tiled cache."""
        _need(q, _F32, "q")
        n = tq * heads * cache.head_dim
        out = torch.empty(max(n, 1), dtype=torch.float32, device=self.device)
        ws = self._flash_ws(tq, past, heads, cache.kv_heads, cache.head_dim)
        _check(self._L.llmtie_flash_attn_t16_ws(self._stream(), _p(q), _n(q), _p(cache.data), _n(cache.data), _p(out),
                                                n, tq, past, heads, cache.kv_heads, cache.head_dim, cache.cap,
                                                scale, int(bool(causal)), _p(ws), _n(ws)))
        return out[:n]

    def t16_append(self, src, src_off, cache: TiledCache16, n, past, value):
        """cache_append_f16 (device.rs:2849) into a tiled cache; value selects V."""
        _need(src, _F32, "src")
        _check(self._L.llmtie_t16_append(self._stream(), _p(src), _n(src), src_off, _p(cache.data), _n(cache.data),
                                         n, cache.kv_heads, cache.head_dim, cache.cap, past, int(bool(value))))

    def t16_rope_cache(self, q, q_off, k, k_off, v, v_off, freq_div, heads, theta, pos, cache: TiledCache16):
        """rope_cache_f16 (device.rs:2915) into a tiled cache."""
        for t, w in ((q, "q"), (k, "k"), (v, "v"), (freq_div, "freq_div")):
            _need(t, _F32, w)
        _check(self._L.llmtie_t16_rope_cache(self._stream(), _p(q), _n(q), q_off, _p(k), _n(k), k_off, _p(v), _n(v),
                                             v_off, _p(freq_div), heads, cache.kv_heads, cache.head_dim,
                                             theta, pos, _p(cache.data), _n(cache.data), cache.cap))

    def t16_grow(self, src: TiledCache16, dst: TiledCache16, live):
        """cache_grow_f16 (device.rs:3152) between tiled caches."""
        _check(self._L.llmtie_t16_grow(self._stream(), _p(src.data), _n(src.data), _p(dst.data), _n(dst.data),
                                       src.kv_heads, src.head_dim, src.cap, dst.cap, live))

    def t16_from_ref(self, k, v, cache: TiledCache16, live):
        """Repack reference-layout f16 caches into a tiled one."""
        _need(k, _H16, "k")
        _need(v, _H16, "v")
        _check(self._L.llmtie_t16_from_ref(self._stream(), _p(k), _n(k), _p(v), _n(v), cache.kv_heads,
                                           cache.head_dim, cache.cap, live, _p(cache.data), _n(cache.data)))

    # ----------------------------------------------------------- producers

    def rope(self, x, off, t, heads, head_dim, theta, first):
        """device.rs:5410."""
        self.rope_scaled(x, off, None, t, heads, head_dim, theta, first)

    def rope_scaled(self, x, off, freq_div, t, heads, head_dim, theta, first):
        """device.rs:5430."""
        _need(x, _F32, "x")
        _need(freq_div, _F32, "freq_div")
        _check(self._L.llmtie_rope(self._stream(), _p(x), _n(x), off, _p(freq_div), t, heads, head_dim,
                                   theta, first))

    def cache_append(self, src, src_off, dst, n, kv_heads, head_dim, cap, past, transposed):
        """device.rs:3013."""
        _need(src, _F32, "src")
        _need(dst, _F32, "dst")
        _check(self._L.llmtie_cache_append(self._stream(), _p(src), _n(src), src_off, _p(dst), _n(dst), n, kv_heads,
                                           head_dim, cap, past, int(bool(transposed))))

    def cache_append_f16(self, src, src_off, dst, n, kv_heads, head_dim, cap, past, transposed):
        """device.rs:2849."""
        _need(src, _F32, "src")
        _need(dst, _H16, "dst")
        _check(self._L.llmtie_cache_append_f16(self._stream(), _p(src), _n(src), src_off, _p(dst), _n(dst), n,
                                               kv_heads, head_dim, cap, past, int(bool(transposed))))

    def rope_cache_f16(self, q, q_off, k, k_off, v, v_off, freq_div, heads, kv_heads, head_dim, theta, pos, kc, vc,
                       cap):
        """device.rs:2915 (the reference passes the projections as (buffer,
        offset) pairs; here as three tensors that may be the same one)."""
        for t, w in ((q, "q"), (k, "k"), (v, "v"), (freq_div, "freq_div")):
            _need(t, _F32, w)
        _need(kc, _H16, "kc")
        _need(vc, _H16, "vc")
        _check(self._L.llmtie_rope_cache_f16(self._stream(), _p(q), _n(q), q_off, _p(k), _n(k), k_off, _p(v), _n(v),
                                             v_off, _p(freq_div), heads, kv_heads, head_dim, theta, pos,
                                             _p(kc), _p(vc), min(_n(kc), _n(vc)), cap))

    def cache_grow(self, src, dst, kv_heads, head_dim, cap, new_cap, live, transposed):
        """device.rs:3086."""
        _need(src, _F32, "src")
        _need(dst, _F32, "dst")
        _check(self._L.llmtie_cache_grow(self._stream(), _p(src), _n(src), _p(dst), _n(dst), kv_heads, head_dim, cap,
                                         new_cap, live, int(bool(transposed))))

    def cache_grow_f16(self, src, dst, kv_heads, head_dim, cap, new_cap, live, transposed):
        """device.rs:3152."""
        _need(src, _H16, "src")
        _need(dst, _H16, "dst")
        _check(self._L.llmtie_cache_grow_f16(self._stream(), _p(src), _n(src), _p(dst), _n(dst), kv_heads, head_dim,
                                             cap, new_cap, live, int(bool(transposed))))

    def kv_q8_append(self, k, k_off, v, v_off, cache: KvCacheQ8, slot, n, past):
        """Quantize n rows of k and v into slot `slot` at positions past.. (new)."""
        _need(k, _F32, "k")
        _need(v, _F32, "v")
        _check(self._L.llmtie_kv_q8_append(self._stream(), _p(k), _n(k), k_off, _p(v), _n(v), v_off, _p(cache.data),
                                           _n(cache.data), cache.slots, slot, n, cache.kv_heads, cache.head_dim,
                                           cache.cap, past))

    def rope_cache_q8(self, q, q_off, k, k_off, v, v_off, freq_div, heads, theta, pos, cache: KvCacheQ8, slot):
        """The Q8_0 twin of rope_cache_f16 (new)."""
        for t, w in ((q, "q"), (k, "k"), (v, "v"), (freq_div, "freq_div")):
            _need(t, _F32, w)
        _check(self._L.llmtie_rope_cache_q8(self._stream(), _p(q), _n(q), q_off, _p(k), _n(k), k_off, _p(v), _n(v),
                                            v_off, _p(freq_div), heads, cache.kv_heads, cache.head_dim,
                                            theta, pos, _p(cache.data), _n(cache.data), cache.slots, slot,
                                            cache.cap))

    # ------------------------------- key ranges and rotary positions by row
    #
    # These calls are a launch or two of a few microseconds, and their host work
    # sets the pace of small ones: checks are one call a tensor, and a result is
    # returned as it was allocated (a view of it costs as much as the allocation).

    def _run(self, fn, *args):
        """A call whose launches go to this Gpu's device, whichever is current."""
        i = self.device.index
        if torch._C._cuda_getDevice() == i:
            status = fn(torch._C._cuda_getCurrentRawStream(i), *args)
        else:
            with torch.cuda.device(self.device):
                status = fn(self._stream(), *args)
        if status:
            _check(status)

    def _on(self, t, dtypes, what, least=0):
        """As _need, on this Gpu's device, and of `least` elements. (An empty
        tensor has no address, which an entry point would take for none given.)"""
        if t is None:
            return
        if t.get_device() != self.device.index or t.dtype not in dtypes or not t.is_contiguous():
            _need(t, dtypes, what)
            raise InvalidArgument(f"{what} is on {t.device}, not on {self.device}")
        if least and t.numel() < least:
            raise SliceOverrun(f"reading to {least} in a buffer of {t.numel()}", (least, t.numel()))

    def key_ranges(self, rows, past=0, starts=None, prefix=None, causal=True, window=0, shared=0) -> KeyRanges:
        """Which keys each of `rows` rows behind `past` positions sees (new; see
        llmtie_key_ranges): documents from `starts` (int32, one more than there
        are), `prefix` leading rows of each that its rows all see, a `window`,
        `shared` leading positions that every row sees."""
        self._on(starts, _I32, "starts", 1)
        self._on(prefix, _I32, "prefix", 1 if starts is None else starts.numel() - 1)
        if rows < 0 or past < 0 or window < 0 or shared < 0:
            raise InvalidArgument("a negative count")
        table = torch.empty((3, rows), dtype=torch.int32, device=self.device)
        pos = torch.empty(rows, dtype=torch.int32, device=self.device)
        self._run(self._L.llmtie_key_ranges, _p(starts), _n(starts), _p(prefix), _n(prefix), rows, past,
                  1 if causal else 0, window, shared, table.data_ptr(), 3 * rows, pos.data_ptr(), rows)
        most = past + rows
        if causal and window and prefix is None:
            most = min(most, window + shared)
        return KeyRanges(table, pos, most)

    def rope_rows(self, x, off, stride, pos, freq_div, t, heads, head_dim, rot_dim, theta, mscale=1.0,
                  interleaved=False, out=None, out_off=0, out_stride=None):
        """Rotary positions by row (new): t rows of `heads` heads at x[off + r *
        stride ..], row r at pos[r] (int32 tensor; an int: pos + r), into `out`
        (f32 or f16; default in place)."""
        if out is None:
            out, out_off, out_stride = x, off, stride
        elif out_stride is None:
            out_stride = heads * head_dim
        self._on(x, _F32, "x")
        self._on(out, _F32 + _H16, "out")
        self._on(freq_div, _F32, "freq_div", rot_dim // 2)
        if isinstance(pos, torch.Tensor):
            self._on(pos, _I32, "pos", t)
            at = pos.data_ptr(), pos.numel(), 0
        else:
            at = None, 0, int(pos)
        if min(off, stride, at[2], t, heads, head_dim, rot_dim, out_off, out_stride) < 0:
            raise InvalidArgument("a negative count")
        self._run(self._L.llmtie_rope_rows, x.data_ptr(), x.numel(), off, stride, out.data_ptr(), out.numel(), out_off,
                  out_stride, 0 if out.dtype is torch.float32 else 1, *at, _p(freq_div), _n(freq_div), t, heads,
                  head_dim, rot_dim, theta, mscale, 1 if interleaved else 0)

    def t16_rope_store(self, q, q_off, k, k_off, v, v_off, stride, pos, slot, index, freq_div, rows, heads, rot_dim,
                       theta, mscale, interleaved, cache: TiledCache16, q_out=None, q_out_off=0, q_out_stride=None):
        """The rotation of q and k with the store of k and v (new): row r of the
        projections (`stride` apart, one stacked tensor or three) to position
        index[r] of slot slot[r] of a tiled cache; q (None: none) into q_out (f32
        or f16; default in place)."""
        self._on(k, _F32, "k")
        self._on(v, _F32, "v")
        f16 = 0
        if q is None:
            q_out_stride = 0
        else:
            self._on(q, _F32, "q")
            if q_out is None:
                q_out, q_out_off, q_out_stride = q, q_off, stride
            else:
                self._on(q_out, _F32 + _H16, "q_out")
                f16 = 0 if q_out.dtype is torch.float32 else 1
                if q_out_stride is None:
                    q_out_stride = heads * cache.head_dim
        for t, what in ((pos, "pos"), (slot, "slot"), (index, "index")):
            self._on(t, _I32, what, rows)
        self._on(freq_div, _F32, "freq_div", rot_dim // 2)
        self._on(cache.data, _H16, "cache")
        if min(q_off, k_off, v_off, stride, rows, heads, rot_dim, q_out_off, q_out_stride) < 0:
            raise InvalidArgument("a negative count")
        self._run(self._L.llmtie_t16_rope_store, _p(q), _n(q), q_off, stride, _p(q_out), _n(q_out), q_out_off,
                  q_out_stride, f16, k.data_ptr(), k.numel(), k_off, stride, v.data_ptr(), v.numel(), v_off, stride,
                  pos.data_ptr(), slot.data_ptr(), index.data_ptr(), rows, _p(freq_div), _n(freq_div), rows, heads,
                  cache.kv_heads, cache.head_dim, rot_dim, theta, mscale, 1 if interleaved else 0,
                  cache.data.data_ptr(), cache.data.numel(), cache.slots, cache.cap)

    def flash_attn_ranges(self, q, q_off, q_stride, cache: TiledCache16, slot, ranges: KeyRanges, tq, past, heads,
                          scale, softcap=0.0, slopes=None):
        """Attention of tq rows (f16) over their key ranges of a slot of a tiled
        cache (new), scores capped (`softcap`) or biased by distance (`slopes`,
        one a head). Returns the f16 context [tq * heads * head_dim]."""
        data, table, hd = cache.data, ranges.table, cache.head_dim
        self._on(q, _H16, "q")
        self._on(data, _H16, "cache")
        self._on(table, _I32, "ranges")
        self._on(slopes, _F32, "slopes", heads)
        if min(q_off, q_stride, slot, tq, past, heads, ranges.max_keys) < 0:
            raise InvalidArgument("a negative count")
        n = tq * heads * hd
        out = torch.empty(n, dtype=torch.float16, device=self.device)
        ws, floats, keys = None, 0, past + tq
        if ranges.max_keys:
            keys = min(ranges.max_keys, keys)
        if keys > 512:  # fewer are never cut
            floats = self._L.llmtie_flash_attn_ranges_workspace(tq, keys, heads, cache.kv_heads, hd)
            if floats:
                try:
                    ws = torch.empty(floats, dtype=torch.float32, device=self.device)
                except torch.OutOfMemoryError:
                    floats = 0  # whole, it needs nothing beside its output
        self._run(self._L.llmtie_flash_attn_ranges_t16, q.data_ptr(), q.numel(), q_off, q_stride, data.data_ptr(),
                  data.numel(), cache.slots, slot, table.data_ptr(), table.numel(), ranges.max_keys, out.data_ptr(), n,
                  tq, past, heads, cache.kv_heads, hd, cache.cap, scale, softcap, _p(slopes), _n(slopes), _p(ws),
                  floats)
        return out

    def attn_decode_ranges(self, q, q_off, q_stride, cache: TiledCache16, tk_dev, slot_dev, max_tk, heads, scale,
                           scratch, lo_dev=None, window=0, shared=0, softcap=0.0, slopes=None, out=None):
        """One token of each of len(tk_dev) sequences over their slots of a tiled
        cache (new): the first `shared` positions and those from max(lo_dev, tk
        - window) on, scores as in flash_attn_ranges. Returns the f32 context."""
        data = cache.data
        self._on(q, _F32, "q")
        self._on(data, _H16, "cache")
        self._on(tk_dev, _I32, "tk")
        self._on(slopes, _F32, "slopes", heads)
        nseq = tk_dev.numel()
        self._on(slot_dev, _I32, "slot", nseq)
        self._on(lo_dev, _I32, "lo", nseq)
        if min(q_off, q_stride, max_tk, heads, window, shared) < 0:
            raise InvalidArgument("a negative count")
        n = nseq * heads * cache.head_dim
        if out is None:
            out = torch.empty(n, dtype=torch.float32, device=self.device)
        else:
            self._on(out, _F32, "out")
        self._run(self._L.llmtie_attn_decode_ranges_t16, q.data_ptr(), q.numel(), q_off, q_stride, data.data_ptr(),
                  data.numel(), cache.slots, tk_dev.data_ptr(), _p(slot_dev), _p(lo_dev), nseq, max_tk, window, shared,
                  heads, cache.kv_heads, cache.head_dim, cache.cap, scale, softcap, _p(slopes), _n(slopes),
                  scratch.handle, out.data_ptr(), out.numel())
        return out if out.numel() == n else out[:n]

    # ------------------------------------------------------ a cache in pages

    def _table(self, table):
        """A page table's address, elements, rows and columns."""
        self._on(table, _I32, "table")
        if table.dim() != 2:
            raise InvalidArgument("a table that is not [rows, pages]")
        return table.data_ptr(), table.numel(), table.shape[0], table.shape[1]

    def _room(self, n, dtype=torch.float32):
        return torch.empty(n, dtype=dtype, device=self.device) if n else None

    def paged_rope_store(self, q, q_off, k, k_off, v, v_off, stride, pos, seq, index, table, freq_div, rows, heads,
                         rot_dim, theta, mscale, interleaved, cache: PagedCache16, q_out=None, q_out_off=0,
                         q_out_stride=None):
        """t16_rope_store into pages (new): row r to position index[r] of the
        sequence whose pages are table[seq[r]]."""
        # (One tensor often: each is looked at once. 32 rows of 32/8/128, 11.7 -> 10.6 us a call.)
        self._on(k, _F32, "k")
        if v is not k:
            self._on(v, _F32, "v")
        f16 = 0
        if q is None:
            q_out_stride = 0
        else:
            if q is not k:
                self._on(q, _F32, "q")
            if q_out is None:
                q_out, q_out_off, q_out_stride = q, q_off, stride
            else:
                self._on(q_out, _F32 + _H16, "q_out")
                f16 = 0 if q_out.dtype is torch.float32 else 1
                if q_out_stride is None:
                    q_out_stride = heads * cache.head_dim
        self._on(pos, _I32, "pos", rows)
        self._on(seq, _I32, "seq", rows)
        if index is not pos:
            self._on(index, _I32, "index", rows)
        self._on(freq_div, _F32, "freq_div", rot_dim // 2)
        self._on(cache.data, _H16, "cache")
        if min(q_off, k_off, v_off, stride, rows, heads, rot_dim, q_out_off, q_out_stride) < 0:
            raise InvalidArgument("a negative count")
        self._run(self._L.llmtie_paged_rope_store, _p(q), _n(q), q_off, stride, _p(q_out), _n(q_out), q_out_off,
                  q_out_stride, f16, k.data_ptr(), k.numel(), k_off, stride, v.data_ptr(), v.numel(), v_off, stride,
                  pos.data_ptr(), seq.data_ptr(), index.data_ptr(), rows, *self._table(table), _p(freq_div),
                  _n(freq_div), rows, heads, cache.kv_heads, cache.head_dim, rot_dim, theta, mscale,
                  1 if interleaved else 0, cache.data.data_ptr(), cache.data.numel(), cache.pages, cache.page)

    def page_plan(self, tk_dev, row_dev, table, heads, cache: PagedCache16, max_tk, starts=None, prefix=None,
                  lo_dev=None, window=0, shared=0) -> PagePlan:
        """The plan of a step's attention for all its layers (new; see
        llmtie_page_plan): len(tk_dev) rows, row r at position tk_dev[r] - 1 of the
        sequence of table[row_dev[r]] (None: table[r]), which sees the first `shared`
        positions and those from max(lo_dev, tk - window) on; rows starts[g] ..
        starts[g + 1] - 1 hold positions below prefix[g] in the same pages."""
        n = tk_dev.numel()
        self._on(tk_dev, _I32, "tk")
        self._on(row_dev, _I32, "row", n)
        self._on(lo_dev, _I32, "lo", n)
        groups = 0
        if starts is not None:
            self._on(starts, _I32, "starts", 1)
            groups = starts.numel() - 1
            if groups and prefix is None:
                raise InvalidArgument("groups without their prefixes")
            self._on(prefix, _I32, "prefix", groups)
        elif prefix is not None:
            raise InvalidArgument("prefixes without their groups")
        _, _, rows, cols = self._table(table)
        if min(max_tk, heads, window, shared) < 0:
            raise InvalidArgument("a negative count")
        kv, hd = cache.kv_heads, cache.head_dim
        size = self._L.llmtie_page_plan_len(n, groups, max_tk, rows, heads, kv)
        plan = torch.empty(size, dtype=torch.int32, device=self.device)
        self._run(self._L.llmtie_page_plan, tk_dev.data_ptr(), _p(row_dev), _p(lo_dev), n, _p(starts), _p(prefix), groups,
                  max_tk, window, shared, rows, cols, cache.page, heads, kv, hd, plan.data_ptr(), size)
        floats = self._L.llmtie_attn_paged_workspace(n, groups, max_tk, rows, heads, kv, hd)
        return PagePlan(plan, tk_dev, table, heads, kv, hd, cache.page, groups, max_tk, floats)

    def attn_decode_paged(self, q, q_off, q_stride, cache: PagedCache16, plan: PagePlan, heads, scale, softcap=0.0,
                          slopes=None, out=None):
        """Attention of the plan's rows over their pages (new), what a group's rows
        share once for all of them, scores as in flash_attn_ranges. Returns the f32
        context [rows * heads * head_dim]."""
        data, hd, kv, nseq = cache.data, cache.head_dim, cache.kv_heads, plan.tk.numel()
        self._on(q, _F32, "q")
        self._on(data, _H16, "cache")
        self._on(plan.data, _I32, "plan")
        self._on(slopes, _F32, "slopes", heads)
        if (heads, kv, hd, cache.page) != (plan.heads, plan.kv_heads, plan.head_dim, plan.page):
            raise InvalidArgument("a plan of other heads or pages")
        if min(q_off, q_stride) < 0:
            raise InvalidArgument("a negative count")
        n = nseq * heads * hd
        if out is None:
            out = torch.empty(n, dtype=torch.float32, device=self.device)
        else:
            self._on(out, _F32, "out")
        ws = self._room(plan.floats)
        self._run(self._L.llmtie_attn_decode_paged, q.data_ptr(), q.numel(), q_off, q_stride, data.data_ptr(),
                  data.numel(), cache.pages, cache.page, *self._table(plan.table), plan.tk.data_ptr(),
                  plan.data.data_ptr(), plan.data.numel(), nseq, plan.groups, plan.max_tk, heads, kv, hd, scale, softcap,
                  _p(slopes), _n(slopes), _p(ws), plan.floats, out.data_ptr(), out.numel())
        return out if out.numel() == n else out[:n]

    def attn_decode_selected(self, q, q_off, q_stride, cache: PagedCache16, table, row_dev, tk_dev, chosen, heads, scale,
                             softcap=0.0, slopes=None, out=None):
        """attn_decode_paged over the pages `chosen` (int32 [rows, kv_heads, count],
        as select_pages returns them) of each row and kv head (new)."""
        data, hd, kv, nseq = cache.data, cache.head_dim, cache.kv_heads, tk_dev.numel()
        self._on(q, _F32, "q")
        self._on(data, _H16, "cache")
        self._on(tk_dev, _I32, "tk")
        self._on(row_dev, _I32, "row", nseq)
        self._on(chosen, _I32, "chosen")
        self._on(slopes, _F32, "slopes", heads)
        if chosen.dim() != 3 or chosen.shape[0] != nseq or chosen.shape[1] != kv:
            raise InvalidArgument(f"pages chosen for {tuple(chosen.shape)}, not for [{nseq}, {kv}, ..]")
        if min(q_off, q_stride, heads) < 0:
            raise InvalidArgument("a negative count")
        count, n = chosen.shape[2], nseq * heads * hd
        if out is None:
            out = torch.empty(n, dtype=torch.float32, device=self.device)
        else:
            self._on(out, _F32, "out")
        pages = self._table(table)
        floats = self._L.llmtie_attn_selected_workspace(nseq, count, cache.page, pages[2], heads, kv, hd)
        ws = self._room(floats)
        self._run(self._L.llmtie_attn_decode_selected, q.data_ptr(), q.numel(), q_off, q_stride, data.data_ptr(),
                  data.numel(), cache.pages, cache.page, *pages, tk_dev.data_ptr(), _p(row_dev),
                  chosen.data_ptr(), chosen.numel(), count, nseq, heads, kv, hd, scale, softcap, _p(slopes), _n(slopes),
                  _p(ws), floats, out.data_ptr(), out.numel())
        return out if out.numel() == n else out[:n]

    def page_bounds(self, cache: PagedCache16, table, row_dev, low_dev, tk_dev, max_new, bounds):
        """The greatest and the least key (f16 `bounds` [pages, kv_heads, 2, head_dim])
        of the pages that hold positions low_dev[r] (None: 0) to tk_dev[r] of each
        row's sequence, over its live positions; max_new of them or so (new)."""
        nseq = tk_dev.numel()
        self._on(cache.data, _H16, "cache")
        self._on(tk_dev, _I32, "tk")
        self._on(row_dev, _I32, "row", nseq)
        self._on(low_dev, _I32, "low", nseq)
        self._on(bounds, _H16, "bounds")
        if max_new < 0:
            raise InvalidArgument("a negative count")
        self._run(self._L.llmtie_page_bounds, cache.data.data_ptr(), cache.data.numel(), cache.pages, cache.page,
                  *self._table(table), _p(row_dev), _p(low_dev), tk_dev.data_ptr(), nseq, max_new, cache.kv_heads,
                  cache.head_dim, bounds.data_ptr(), bounds.numel())

    def select_pages(self, q, q_off, q_stride, bounds, table, row_dev, tk_dev, max_tk, heads, page, count, first=1,
                     last=1):
        """The `count` pages that each row and kv head attends (new): the first `first`
        and `last` last ones and those whose `bounds` (page_bounds) allow the largest
        product with one of its heads. Returns int32 [rows, kv_heads, count], rising,
        -1 behind the last."""
        nseq = tk_dev.numel()
        self._on(q, _F32, "q")
        self._on(bounds, _H16, "bounds")
        self._on(tk_dev, _I32, "tk")
        self._on(row_dev, _I32, "row", nseq)
        if bounds.dim() != 4 or bounds.shape[2] != 2:
            raise InvalidArgument("bounds that are not [pages, kv_heads, 2, head_dim]")
        pages, kv, _, hd = bounds.shape
        if min(q_off, q_stride, max_tk, heads, page, count, first, last) < 0:
            raise InvalidArgument("a negative count")
        chosen = torch.empty((nseq, kv, count), dtype=torch.int32, device=self.device)
        room = self._L.llmtie_select_pages_workspace(nseq, max_tk, page, count, kv)
        ws = self._room(room, torch.float64)
        self._run(self._L.llmtie_select_pages, q.data_ptr(), q.numel(), q_off, q_stride, bounds.data_ptr(),
                  bounds.numel(), pages, page, *self._table(table), tk_dev.data_ptr(), _p(row_dev), nseq, max_tk, heads,
                  kv, hd, count, first, last, _p(ws), room, chosen.data_ptr(), chosen.numel())
        return chosen
