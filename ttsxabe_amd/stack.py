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
the slots of tiled caches. `LlamaPages` does so over pages, which sequences that
begin alike share.
"""
from __future__ import annotations

from collections import Counter

import numpy as np
import torch

from .gpu import CacheOverrun, DecodeScratch, Gpu, InvalidArgument, PagedCache16, TiledCache16, rope_scaling

PLAN_GROUPS = 1024  # that Gpu.page_plan takes


def _no_selection(cfg):
    if getattr(cfg, "select", None) is not None:
        raise ValueError("a configuration that selects pages, which LlamaPages attends")


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
        _no_selection(cfg)
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


class _Sequences:
    """What several sequences of one stack at once have in common, wherever their keys lie."""

    def __init__(self, gpu: Gpu, cfg, weights: dict, slots: int, cap: int):
        self.g, self.cfg, self.slots, self.cap = gpu, cfg, slots, cap
        dev = gpu.device
        w = {k: torch.from_numpy(np.ascontiguousarray(v)).to(dev) for k, v in weights.items()}
        for l in range(cfg.layers):  # q, k and v in one product, rows the rotation and the stores read as they are
            w[f"{l}.wqkv"] = torch.cat([w.pop(f"{l}.wq"), w.pop(f"{l}.wk"), w.pop(f"{l}.wv")])
        self.w = w
        self.packed = None  # the keys of the prompts being packed, one layer at a time
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

    def _check(self, slots, new, ids, length=None):
        # (An id past the embedding ends the process from the device.)
        length = self.length if length is None else length
        vocab = len(self.w["embed"])
        if ids and not (min(ids) >= 0 and max(ids) < vocab):
            raise InvalidArgument(f"a token that is not one of {vocab}")
        if len(set(slots)) < len(slots) or any(not 0 <= s < self.slots for s in slots):
            raise InvalidArgument(f"slots {slots} of {self.slots}")
        for s, n in zip(slots, new):
            if n < 1:
                raise InvalidArgument("a sequence without tokens")
            if length[s] + n > self.cap:
                raise CacheOverrun(f"appending at {length[s] + n} to a cache with room for {self.cap}",
                                   (length[s] + n, self.cap))

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

    def _logits(self, h):
        return self._norm(h, self.w["norm"]) @ self.w["lm_head"].T

    def _parts(self, qkv, q):
        """A stacked projection as the stores' first arguments (q: whether it is rotated too)."""
        qd, kd = self.cfg.heads * self.cfg.head_dim, self.cfg.kv_heads * self.cfg.head_dim
        return qkv if q else None, 0, qkv, qd, qkv, qd + kd, qd + 2 * kd

    def _store(self, qkv, q, pos, slot, index, cache, q_out):
        self.g.t16_rope_store(*self._parts(qkv, q), pos, slot, index, self.div, len(pos), self.cfg.heads, self.rot,
                              self.theta, self.mscale, self.inter, cache, q_out=q_out)

    def _ranges(self, lens):
        """Which keys the rows of packed prompts see; None where they go one by one."""
        g, n = self.g, sum(lens)
        starts = self._ints(np.concatenate([[0], np.cumsum(lens)]).tolist())
        if self.shared and self.window:
            # Each document's own leading positions stay seen: a range of keys
            # holds one run of them only, so documents longer than the window
            # and these go one by one.
            if max(lens) > self.window + self.shared:
                return None if len(lens) > 1 else g.key_ranges(n, 0, None, None, True, self.window, self.shared)
            return g.key_ranges(n, 0, starts, None, True, 0, 0)
        return g.key_ranges(n, 0, starts, None, True, self.window, 0)

    def _pack(self, tokens, lens, r, keep):
        """Logits of packed prompts' last tokens, attended in a cache of their own; keep(l, qkv) stores a layer's keys
        where they stay."""
        c, g, n = self.cfg, self.g, len(tokens)
        if self.packed is None or self.packed.cap < n:
            self.packed = TiledCache16(c.kv_heads, c.head_dim, max(256, 1 << (n - 1).bit_length()), device=g.device,
                                       zero=False)
        row = torch.arange(n, dtype=torch.int32, device=g.device)
        zero = torch.zeros_like(row)
        q = torch.empty(n * c.heads * c.head_dim, dtype=torch.float16, device=g.device)

        def attend(l, qkv):
            self._store(qkv, True, r.pos, zero, row, self.packed, q)
            keep(l, qkv)
            return g.flash_attn_ranges(q, 0, c.heads * c.head_dim, self.packed, 0, r, n, 0, c.heads, self.scale,
                                       **self.scores)

        last = torch.tensor(np.cumsum(lens) - 1, device=g.device)
        return self._logits(self._layers(torch.tensor(tokens, device=g.device), attend)[last])


class LlamaBatch(_Sequences):
    """Up to `slots` sequences of `cap` positions side by side. Beside the
    geometry `cfg` may hold `rope_interleaved` (weights for pairs (2i, 2i + 1), as
    a GGUF stores them), `rope_dim` (rotated dims of a head, 0: all),
    `rope_scaling` ((kind, factor, original positions), see gpu.rope_scaling),
    `softcap`, `window` with `shared` leading positions kept, and `slopes` (a
    distance bias a head)."""

    def __init__(self, gpu: Gpu, cfg, weights: dict, slots: int, cap: int):
        _no_selection(cfg)
        super().__init__(gpu, cfg, weights, slots, cap)
        self.cache = [TiledCache16(cfg.kv_heads, cfg.head_dim, cap, device=gpu.device, slots=slots)
                      for _ in range(cfg.layers)]
        self.scratch = DecodeScratch()

    def prefill(self, prompts, slots) -> torch.Tensor:
        """Logits [len(prompts), vocab] of the prompts' last tokens; prompt i begins a sequence in slots[i] (what was
        there is dropped)."""
        lens = [len(p) for p in prompts]
        if len(slots) != len(prompts) or not prompts:
            raise InvalidArgument("a slot for each prompt")
        tokens = [int(t) for p in prompts for t in p]
        begun = [0 if s in set(slots) else n for s, n in enumerate(self.length)]
        self._check(slots, lens, tokens, begun)
        self.length = begun
        r = self._ranges(lens)
        if r is None:
            return torch.cat([self.prefill([p], [s]) for p, s in zip(prompts, slots)])
        slot = self._ints(np.repeat(slots, lens).tolist())
        out = self._pack(tokens, lens, r,
                         lambda l, qkv: self._store(qkv, False, r.pos, slot, r.pos, self.cache[l], None))
        for s, m in zip(slots, lens):
            self.length[s] = m
        return out

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
        return self._logits(h)


class LlamaPages(_Sequences):
    """Up to `slots` sequences of up to `cap` positions over one pool of `pages` pages of `page` positions a layer
    (a power of two from 32): each holds the pages of its length, and sequences begun behind another share its full
    pages, which a step attends once for all of them. `cfg` as LlamaBatch's; its `select` ((count, first, last), no
    window beside it) has a step's sequences of more pages than `count` attend so many of them, the first and last
    ones and those whose keys' bounds allow the largest products."""

    def __init__(self, gpu: Gpu, cfg, weights: dict, slots: int, cap: int, pages: int, page: int = 64):
        self.select = getattr(cfg, "select", None)
        if self.select is not None and getattr(cfg, "window", 0):
            raise ValueError("a configuration that selects pages behind a window")
        super().__init__(gpu, cfg, weights, slots, cap)
        dev = gpu.device
        self.page, self.cache = page, [PagedCache16(cfg.kv_heads, cfg.head_dim, pages, page, device=dev)
                                       for _ in range(cfg.layers)]
        self.bounds = None
        if self.select is not None:
            self.bounds = [torch.zeros(pages, cfg.kv_heads, 2, cfg.head_dim, dtype=torch.float16, device=dev)
                           for _ in range(cfg.layers)]
        self.spare = list(range(pages - 1, -1, -1))  # pages that nobody holds
        self.held = [0] * pages                      # sequences that hold a page
        self.own = [[] for _ in range(slots)]        # pages of each sequence, in order
        self.table = torch.full((slots, (cap + page - 1) // page), -1, dtype=torch.int32, device=dev)

    def free(self, slots):
        """Ends the sequences in `slots`."""
        self._check(slots, [], [])
        for s in slots:
            for p in self.own[s]:
                self.held[p] -= 1
                if not self.held[p]:
                    self.spare.append(p)
            self.own[s], self.length[s] = [], 0

    def _take(self, need):
        """Pages for need[s] more positions of each slot s (all of them, or none)."""
        more = {s: (self.length[s] + n + self.page - 1) // self.page - len(self.own[s]) for s, n in need.items()}
        if sum(more.values()) > len(self.spare):
            raise CacheOverrun(f"{sum(more.values())} pages of {len(self.spare)}", (sum(more.values()), len(self.spare)))
        for s, n in more.items():
            for _ in range(n):
                p = self.spare.pop()
                self.held[p] = 1
                self.own[s].append(p)

    def _show(self, slots):
        """The slots' rows of the table on the device."""
        wide = self.table.shape[1]
        self.table[torch.tensor(list(slots), device=self.g.device)] = self._ints(
            [self.own[s] + [-1] * (wide - len(self.own[s])) for s in slots])

    def _keep(self, l, qkv, q, pos, row, q_out=None):
        c = self.cfg
        self.g.paged_rope_store(*self._parts(qkv, q), pos, row, pos, self.table, self.div, len(pos), c.heads, self.rot,
                                self.theta, self.mscale, self.inter, self.cache[l], q_out=q_out)

    def _bound(self, l, row, low, tk, new):
        if self.bounds is not None:
            self.g.page_bounds(self.cache[l], self.table, row, low, tk, new, self.bounds[l])

    def prefill(self, prompts, slots, behind=None) -> torch.Tensor:
        """Logits [len(prompts), vocab] of the prompts' last tokens; prompt i begins a sequence in slots[i] (what was
        there is dropped), behind all positions of the sequence in slot `behind` if that is given."""
        lens = [len(p) for p in prompts]
        if len(slots) != len(prompts) or not prompts:
            raise InvalidArgument("a slot for each prompt")
        if behind is not None and (not 0 <= behind < self.slots or behind in slots or not self.length[behind]):
            raise InvalidArgument(f"sequences behind slot {behind}")
        tokens = [int(t) for p in prompts for t in p]
        past = 0 if behind is None else self.length[behind]
        self._check(slots, lens, tokens, [past] * self.slots)
        lead = [] if behind is None else self.own[behind][:past // self.page]
        ending = Counter(p for s in slots for p in self.own[s])
        freed = sum(self.held[p] == n for p, n in ending.items())
        need = sum((past + n + self.page - 1) // self.page - len(lead) for n in lens)
        if need > len(self.spare) + freed:
            raise CacheOverrun(f"{need} pages of {len(self.spare) + freed}", (need, len(self.spare) + freed))
        self.free(slots)
        try:
            return self._fill(prompts, lens, slots, tokens, behind, past, lead)
        except Exception:  # (of keys that were not all stored there is nothing to go on from)
            self.free(slots)
            raise

    def _fill(self, prompts, lens, slots, tokens, behind, past, lead):
        """The prompts' pages (`lead` ones of the `past` positions that they follow before them) and their pass."""
        for s in slots:
            self.own[s] = list(lead)
            for p in lead:
                self.held[p] += 1
            self.length[s] = len(lead) * self.page
        self._take({s: past + n - self.length[s] for s, n in zip(slots, lens)})
        self._show(slots)
        if past % self.page:  # the page that is not full is each one's own
            old = self.own[behind][len(lead)]
            new = torch.tensor([self.own[s][len(lead)] for s in slots], device=self.g.device)
            for c in self.cache:
                c.data.view(c.pages, -1)[new] = c.data.view(c.pages, -1)[old].clone()
        for s, n in zip(slots, lens):
            self.length[s] = past + n
        if behind is None:
            return self._begin(prompts, lens, slots, tokens)
        c, g, n = self.cfg, self.g, len(tokens)
        at = [past + j for m in lens for j in range(m)]
        pos, row = self._ints(at), self._ints(np.repeat(slots, lens).tolist())
        ends, first = self._ints([past + m for m in lens]), self._ints([past] * len(lens))
        rows = self._ints(list(slots))
        tk = pos + 1
        # (As rows of a table of these sequences alone: there are then more rows than sequences.)
        few, which = self.table[rows.long()], self._ints(np.repeat(np.arange(len(slots)), lens).tolist())
        plan = g.page_plan(tk, which, few, c.heads, self.cache[0], past + max(lens), starts=self._ints([0, n]),
                           prefix=self._ints([len(lead) * self.page]), window=self.window, shared=self.shared)
        q = torch.empty(n * c.heads * c.head_dim, dtype=torch.float32, device=g.device)

        def attend(l, qkv):
            self._keep(l, qkv, True, pos, row, q)
            self._bound(l, rows, first, ends, max(lens))
            return g.attn_decode_paged(q, 0, c.heads * c.head_dim, self.cache[l], plan, c.heads, self.scale, **self.scores)

        last = torch.tensor(np.cumsum(lens) - 1, device=g.device)
        return self._logits(self._layers(torch.tensor(tokens, device=g.device), attend)[last])

    def _begin(self, prompts, lens, slots, tokens):
        r = self._ranges(lens)
        if r is None:
            return torch.cat([self._begin([p], [len(p)], [s], [int(t) for t in p]) for p, s in zip(prompts, slots)])
        row, rows, ends = self._ints(np.repeat(slots, lens).tolist()), self._ints(list(slots)), self._ints(lens)

        def keep(l, qkv):
            self._keep(l, qkv, False, r.pos, row)
            self._bound(l, rows, None, ends, max(lens))

        return self._pack(tokens, lens, r, keep)

    def _groups(self, slots):
        """`slots` in an order in which sequences that share pages follow one another: the order, each group's
        first row and the one behind the last, and the positions that its rows share."""
        order = sorted(range(len(slots)), key=lambda i: self.own[slots[i]])
        starts, prefix = [], []
        for i, x in enumerate(order):
            own = self.own[slots[x]]
            if starts:
                head = self.own[slots[order[starts[-1]]]]
                n = next((k for k, (a, b) in enumerate(zip(head, own)) if a != b), min(len(head), len(own)))
                had = prefix[-1] // self.page if i - starts[-1] > 1 else n
                if n and 2 * n >= had:  # (else it would take more than half of what the others share)
                    prefix[-1] = min(had, n) * self.page
                    continue
            starts.append(i)
            prefix.append(0)
        # Sequences that share nothing side by side as one group, and no more groups than a plan takes.
        kept = [i for i in range(len(starts)) if prefix[i] or not i or prefix[i - 1]][:PLAN_GROUPS]
        starts, prefix = [starts[i] for i in kept], [prefix[i] for i in kept]
        if len(kept) == PLAN_GROUPS:
            prefix[-1] = 0
        return order, starts + [len(slots)], prefix

    def step(self, ids, slots) -> torch.Tensor:
        """Logits [len(ids), vocab] after one more token of each of the sequences in `slots`."""
        c, g = self.cfg, self.g
        if len(ids) != len(slots) or not slots:
            raise InvalidArgument("a token for each slot")
        ids = [int(t) for t in ids]
        self._check(slots, [1] * len(slots), ids)
        if any(not self.length[s] for s in slots):
            raise InvalidArgument("a step of a sequence that is not begun")
        more = [s for s in slots if self.length[s] == len(self.own[s]) * self.page]
        self._take({s: 1 for s in more})
        if more:
            self._show(more)
        order, starts, prefix = self._groups(slots)
        to = [slots[i] for i in order]
        at = [self.length[s] for s in to]
        pos, row, tk = self._ints(at), self._ints(to), self._ints([p + 1 for p in at])
        q = torch.empty(len(ids) * c.heads * c.head_dim, dtype=torch.float32, device=g.device)
        width, most = c.heads * c.head_dim, max(at) + 1
        few = self.select is not None and (most + self.page - 1) // self.page > self.select[0]
        if not few:
            sharing = any(prefix)
            plan = g.page_plan(tk, row, self.table, c.heads, self.cache[0], most,
                               starts=self._ints(starts) if sharing else None,
                               prefix=self._ints(prefix) if sharing else None, window=self.window, shared=self.shared)

        def attend(l, qkv):
            self._keep(l, qkv, True, pos, row, q)
            self._bound(l, row, pos, tk, 1)
            if not few:
                return g.attn_decode_paged(q, 0, width, self.cache[l], plan, c.heads, self.scale, **self.scores)
            chosen = g.select_pages(q, 0, width, self.bounds[l], self.table, row, tk, most, c.heads, self.page,
                                    *self.select)
            return g.attn_decode_selected(q, 0, width, self.cache[l], self.table, row, tk, chosen, c.heads, self.scale,
                                          **self.scores)

        h = self._layers(torch.tensor([ids[i] for i in order], device=g.device), attend)
        for s in slots:
            self.length[s] += 1
        back = torch.empty(len(order), dtype=torch.long)
        back[torch.tensor(order)] = torch.arange(len(order))
        return self._logits(h)[back.to(g.device)]
