"""A Llama decoder stack around the attention path, on one MI355X.

The caller side of the path as the reference's chat model arranges it
(crates/llmtie-chat/src/model.rs:700-1175): per layer RMSNorm, the q/k/v
projections, RoPE with the K/V cache write, attention, the output projection
and residual, then RMSNorm and the SwiGLU feed-forward; a final RMSNorm and
the LM head. The projections, norms and SwiGLU are plain torch f32 ops here
(plumbing); RoPE, the cache writes, cache growth and attention go through this
library, which is the part under test. Weights come from the caller (random,
for the argmax check against the CPU restatement of the same stack).

The cache grows like the reference's: to the next power of two of what is
needed, at least 256 positions (model.rs:703-721), copying the live prefix.

`LlamaBatch` (no counterpart in the reference, which steps its sequences one
by one) runs several sequences of the same stack at once: prompts packed into
one pass, each a document of its own, and one token of all of them a step, over
the slots of tiled caches.
"""
from __future__ import annotations

import numpy as np
import torch

from .gpu import CacheOverrun, DecodeScratch, Gpu, InvalidArgument, TiledCache16, rope_scaling


class LlamaStack:
    """`layout`: "reference" (K [kv][cap][hd] + V [kv][hd][cap] f16, the
    reference's cache) or "tiled" (the fragment-order cache). Plain scores, and
    whole heads rotated in halves at unscaled positions: a configuration that asks for
    others is refused."""

    def __init__(self, gpu: Gpu, cfg, weights: dict, layout: str = "reference"):
        if layout not in ("reference", "tiled"):
            raise ValueError(f"unknown cache layout {layout!r}")
        kind, factor, _ = getattr(cfg, "rope_scaling", None) or ("none", 1.0, 0)
        for what, has in (("interleaved rotary weights", getattr(cfg, "rope_interleaved", False)),
                          ("capped scores", getattr(cfg, "softcap", 0.0)),
                          ("a window", getattr(cfg, "window", 0)),
                          ("biased scores", getattr(cfg, "slopes", None) is not None),
                          ("partly rotated heads", (getattr(cfg, "rope_dim", 0) or cfg.head_dim) != cfg.head_dim),
                          ("scaled rotary positions", kind != "none" and factor != 1.0)):
            if has:
                raise ValueError(f"a configuration with {what}, which LlamaBatch computes")
        self.g, self.cfg, self.layout = gpu, cfg, layout
        dev = gpu.device
        self.w = {k: torch.from_numpy(np.ascontiguousarray(v)).to(dev) for k, v in weights.items()}
        self.past = 0
        self.cap = 0
        self.kc, self.vc, self.tc = [], [], []
        self.scratch = DecodeScratch()

    def _grow(self, need: int):
        if need <= self.cap:
            return
        c = self.cfg
        want = max(256, 1 << (need - 1).bit_length())
        kvd = c.kv_heads * c.head_dim
        for l in range(c.layers):
            if self.layout == "tiled":
                t = TiledCache16(c.kv_heads, c.head_dim, want, device=self.g.device)
                if self.past:
                    self.g.t16_grow(self.tc[l], t, self.past)
                if l < len(self.tc):
                    self.tc[l] = t
                else:
                    self.tc.append(t)
            else:
                k = torch.zeros(want * kvd, dtype=torch.float16, device=self.g.device)
                v = torch.zeros(want * kvd, dtype=torch.float16, device=self.g.device)
                if self.past:
                    self.g.cache_grow_f16(self.kc[l], k, c.kv_heads, c.head_dim, self.cap, want, self.past, False)
                    self.g.cache_grow_f16(self.vc[l], v, c.kv_heads, c.head_dim, self.cap, want, self.past, True)
                if l < len(self.kc):
                    self.kc[l], self.vc[l] = k, v
                else:
                    self.kc.append(k)
                    self.vc.append(v)
        self.cap = want

    def _norm(self, x, w):
        """crates/llmtie-dsp/src/rope.rs:16-28."""
        return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + self.cfg.eps) * w

    def forward(self, ids) -> torch.Tensor:
        """Logits [vocab] of the last of `ids`, which extend the cache."""
        c, g, w = self.cfg, self.g, self.w
        n, past, hd = len(ids), self.past, c.head_dim
        self._grow(past + n)
        scale = float(np.float32(hd) ** np.float32(-0.5))
        fd = w.get("rope_freqs")  # Llama-3 per-frequency RoPE divisors, when the checkpoint has them
        h = w["embed"][torch.as_tensor(list(ids), device=g.device)]
        for l in range(c.layers):
            x = self._norm(h, w[f"{l}.attn_norm"])
            q = (x @ w[f"{l}.wq"].T).contiguous().view(-1)
            k = (x @ w[f"{l}.wk"].T).contiguous().view(-1)
            v = (x @ w[f"{l}.wv"].T).contiguous().view(-1)
            if self.layout == "tiled":
                t = self.tc[l]
                if n == 1:
                    g.t16_rope_cache(q, 0, k, 0, v, 0, fd, c.heads, c.theta, past, t)
                    ctx = g.attn_decode_t16(q, t, c.heads, past + 1, scale, False, self.scratch)
                else:
                    g.rope_scaled(q, 0, fd, n, c.heads, hd, c.theta, past)
                    g.rope_scaled(k, 0, fd, n, c.kv_heads, hd, c.theta, past)
                    g.t16_append(k, 0, t, n, past, False)
                    g.t16_append(v, 0, t, n, past, True)
                    ctx = g.flash_attn_t16(q, t, n, past, c.heads, scale, True)
            else:
                kc, vc = self.kc[l], self.vc[l]
                if n == 1:
                    g.rope_cache_f16(q, 0, k, 0, v, 0, fd, c.heads, c.kv_heads, hd, c.theta, past, kc, vc,
                                     self.cap)
                    ctx = g.attn_decode_f16(q, kc, vc, c.heads, c.kv_heads, hd, past + 1, self.cap, scale, False,
                                            self.scratch)
                else:
                    g.rope_scaled(q, 0, fd, n, c.heads, hd, c.theta, past)
                    g.rope_scaled(k, 0, fd, n, c.kv_heads, hd, c.theta, past)
                    g.cache_append_f16(k, 0, kc, n, c.kv_heads, hd, self.cap, past, False)
                    g.cache_append_f16(v, 0, vc, n, c.kv_heads, hd, self.cap, past, True)
                    ctx = g.flash_attn_f16(q, kc, vc, n, past, c.heads, c.kv_heads, hd, self.cap, scale, True)
            h = h + ctx.view(n, -1) @ w[f"{l}.wo"].T
            x = self._norm(h, w[f"{l}.ffn_norm"])
            h = h + (torch.nn.functional.silu(x @ w[f"{l}.wg"].T) * (x @ w[f"{l}.wu"].T)) @ w[f"{l}.wd"].T
        self.past += n
        return (self._norm(h[-1:], w["norm"]) @ w["lm_head"].T)[0]


class LlamaBatch:
    """Up to `slots` sequences of `cap` positions side by side. Beside the
    geometry `cfg` may hold `rope_interleaved` (weights for pairs (2i, 2i + 1), as
    a GGUF stores them), `rope_dim` (rotated dims of a head, 0: all),
    `rope_scaling` ((kind, factor, original positions), see gpu.rope_scaling),
    `softcap`, `window` with `shared` leading positions kept, and `slopes` (a
    distance bias a head)."""

    def __init__(self, gpu: Gpu, cfg, weights: dict, slots: int, cap: int):
        self.g, self.cfg, self.slots, self.cap = gpu, cfg, slots, cap
        dev = gpu.device
        w = {k: torch.from_numpy(np.ascontiguousarray(v)).to(dev) for k, v in weights.items()}
        for l in range(cfg.layers):  # q, k and v in one product, rows the rotation and the stores read as they are
            w[f"{l}.wqkv"] = torch.cat([w.pop(f"{l}.wq"), w.pop(f"{l}.wk"), w.pop(f"{l}.wv")])
        self.w = w
        self.cache = [TiledCache16(cfg.kv_heads, cfg.head_dim, cap, device=dev, slots=slots) for _ in range(cfg.layers)]
        self.packed = None  # the keys of the prompts being packed, one layer at a time
        self.scratch = DecodeScratch()
        self.length = [0] * slots
        self.rot = getattr(cfg, "rope_dim", 0) or cfg.head_dim
        kind, factor, original = getattr(cfg, "rope_scaling", None) or ("none", 1.0, 8192)
        div, self.theta, self.mscale = rope_scaling(self.rot, cfg.theta, kind, factor, original, device=dev)
        freqs = w.get("rope_freqs")  # a checkpoint's own divisors, beside the scaling's
        self.div = freqs if div is None else div if freqs is None else div * freqs
        self.inter = bool(getattr(cfg, "rope_interleaved", False))
        self.window, self.shared = getattr(cfg, "window", 0), getattr(cfg, "shared", 0)
        slopes = getattr(cfg, "slopes", None)
        self.scores = dict(softcap=float(getattr(cfg, "softcap", 0.0)),
                           slopes=None if slopes is None else torch.as_tensor(slopes, dtype=torch.float32, device=dev))
        self.scale = float(np.float32(cfg.head_dim) ** np.float32(-0.5))

    def _ints(self, v):
        return torch.tensor(v, dtype=torch.int32, device=self.g.device)

    def _check(self, slots, new, ids):
        # (An id past the embedding ends the process from the device.)
        vocab = len(self.w["embed"])
        if ids and not (min(ids) >= 0 and max(ids) < vocab):
            raise InvalidArgument(f"a token that is not one of {vocab}")
        if len(set(slots)) < len(slots) or any(not 0 <= s < self.slots for s in slots):
            raise InvalidArgument(f"slots {slots} of {self.slots}")
        for s, n in zip(slots, new):
            if n < 1:
                raise InvalidArgument("a sequence without tokens")
            if self.length[s] + n > self.cap:
                raise CacheOverrun(f"appending at {self.length[s] + n} to a cache with room for {self.cap}",
                                   (self.length[s] + n, self.cap))

    def _norm(self, x, w):
        return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + self.cfg.eps) * w

    def _layers(self, ids, attend):
        """The hidden rows of `ids` [n] after the last layer; attend(l, qkv [n, ..]) is a layer's context."""
        c, w = self.cfg, self.w
        h = w["embed"][ids]
        for l in range(c.layers):
            qkv = (self._norm(h, w[f"{l}.attn_norm"]) @ w[f"{l}.wqkv"].T).contiguous()
            h = h + attend(l, qkv).view(len(ids), -1).float() @ w[f"{l}.wo"].T
            x = self._norm(h, w[f"{l}.ffn_norm"])
            h = h + (torch.nn.functional.silu(x @ w[f"{l}.wg"].T) * (x @ w[f"{l}.wu"].T)) @ w[f"{l}.wd"].T
        return h

    def _store(self, qkv, q, pos, slot, index, cache, q_out):
        c = self.cfg
        qd, kd = c.heads * c.head_dim, c.kv_heads * c.head_dim
        self.g.t16_rope_store(qkv if q else None, 0, qkv, qd, qkv, qd + kd, qd + 2 * kd, pos, slot, index, self.div,
                              len(pos), c.heads, self.rot, self.theta, self.mscale, self.inter, cache, q_out=q_out)

    def prefill(self, prompts, slots) -> torch.Tensor:
        """Logits [len(prompts), vocab] of the prompts' last tokens; prompt i begins a sequence in slots[i] (what was
        there is dropped)."""
        c, g = self.cfg, self.g
        lens = [len(p) for p in prompts]
        if len(slots) != len(prompts) or not prompts:
            raise InvalidArgument("a slot for each prompt")
        tokens = [int(t) for p in prompts for t in p]
        before = self.length
        self.length = [0 if s in set(slots) else n for s, n in enumerate(before)]
        try:
            self._check(slots, lens, tokens)
        except Exception:
            self.length = before
            raise
        n = sum(lens)
        starts = np.concatenate([[0], np.cumsum(lens)]).tolist()
        r = g.key_ranges(n, 0, self._ints(starts), None, True, self.window, 0)
        if self.shared and self.window:
            # Each document's own leading positions stay seen: a range of keys
            # holds one run of them only, so documents longer than the window
            # and these go one by one.
            if max(lens) > self.window + self.shared:
                if len(prompts) > 1:
                    return torch.cat([self.prefill([p], [s]) for p, s in zip(prompts, slots)])
                r = g.key_ranges(n, 0, None, None, True, self.window, self.shared)
            else:
                r = g.key_ranges(n, 0, self._ints(starts), None, True, 0, 0)
        if self.packed is None or self.packed.cap < n:
            self.packed = TiledCache16(c.kv_heads, c.head_dim, max(256, 1 << (n - 1).bit_length()), device=g.device,
                                       zero=False)
        row = torch.arange(n, dtype=torch.int32, device=g.device)
        zero = torch.zeros_like(row)
        slot = self._ints(np.repeat(slots, lens).tolist())
        q = torch.empty(n * c.heads * c.head_dim, dtype=torch.float16, device=g.device)

        def attend(l, qkv):
            self._store(qkv, True, r.pos, zero, row, self.packed, q)
            self._store(qkv, False, r.pos, slot, r.pos, self.cache[l], None)
            return g.flash_attn_ranges(q, 0, c.heads * c.head_dim, self.packed, 0, r, n, 0, c.heads, self.scale,
                                       **self.scores)

        h = self._layers(torch.tensor(tokens, device=g.device), attend)[torch.tensor(starts[1:], device=g.device) - 1]
        for s, m in zip(slots, lens):
            self.length[s] = m
        return self._norm(h, self.w["norm"]) @ self.w["lm_head"].T

    def step(self, ids, slots) -> torch.Tensor:
        """Logits [len(ids), vocab] after one more token of each of the sequences in `slots`."""
        c, g = self.cfg, self.g
        if len(ids) != len(slots) or not slots:
            raise InvalidArgument("a token for each slot")
        ids = [int(t) for t in ids]
        self._check(slots, [1] * len(slots), ids)
        at = [self.length[s] for s in slots]
        pos, slot, tk = self._ints(at), self._ints(list(slots)), self._ints([p + 1 for p in at])
        q = torch.empty(len(ids) * c.heads * c.head_dim, dtype=torch.float32, device=g.device)

        def attend(l, qkv):
            self._store(qkv, True, pos, slot, pos, self.cache[l], q)
            return g.attn_decode_ranges(q, 0, c.heads * c.head_dim, self.cache[l], tk, slot, max(at) + 1, c.heads,
                                        self.scale, self.scratch, window=self.window, shared=self.shared, **self.scores)

        h = self._layers(torch.tensor(ids, device=g.device), attend)
        for s in slots:
            self.length[s] += 1
        return self._norm(h, self.w["norm"]) @ self.w["lm_head"].T
