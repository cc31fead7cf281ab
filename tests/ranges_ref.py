"""Plain 64-bit implementations of attention over key ranges and of rotary
positions by row, with the error that the kernels' arithmetic allows (test
infrastructure).

Error of a context, from the steps that round (u = 2^-24 is half a step of f32,
h = 2^-11 of f16):
  scores   an f32 sum of hd exact products, off by at most hd u sum|q k|
           times the scale (the decode's q is a sum of two f16: 2^-22 of it and
           2^-25 more), then the cap (a tanh of values up to c, off by a few
           u c), the bias and the base-2 exponent, a few u of their values:
             d_j = u (hd + 8) scale sum|q k| + 16 u c + 8 u (|s_j| + bias_j)
           which moves p_j by the factor 1 +- d_j, and the sum of all by their mean;
  weights  p_j rounded for the product: h (prompts) or 2^-22 (decode) of each, and
           half a step of f16's smallest, 2^-25 of the largest weight; the prompts'
           normaliser is the sum of the rounded ones, as far off as its terms;
  sums     f32 sums over n keys: n u of sum p|v|, and as much of the normaliser;
  output   h (f16) or u (f32) of the value, and f16's 2^-25.
"""
import math

import numpy as np
import torch

from tiled import t16_index

U, H = 2.0 ** -24, 2.0 ** -11


def tile(k, v):
    """K, V [slots, kv, cap, hd] (f16) as a tiled cache buffer; positions past cap hold zeros."""
    slots, kv, cap, hd = k.shape
    nb = (cap + 31) // 32
    kk = torch.zeros(slots, kv, nb * 32, hd, dtype=torch.float16)
    vv = torch.zeros_like(kk)
    kk[:, :, :cap], vv[:, :, :cap] = k, v
    kk, vv = kk.view(slots, kv, nb, 32, hd), vv.view(slots, kv, nb, 32, hd)
    a, b, c, d = (torch.from_numpy(np.array(x)).long() for x in t16_index(hd))
    return torch.stack([kk[:, :, :, a, b], vv[:, :, :, c, d]], 3).reshape(-1)


def untile(data, slots, kv, hd, cap):
    nb = (cap + 31) // 32
    x = data.view(slots, kv, nb, 2, 32 * hd)
    a, b, c, d = (torch.from_numpy(np.array(x)).long() for x in t16_index(hd))
    k = torch.zeros(slots, kv, nb, 32, hd, dtype=data.dtype)
    v = torch.zeros_like(k)
    k[:, :, :, a, b], v[:, :, :, c, d] = x[:, :, :, 0], x[:, :, :, 1]
    return k.view(slots, kv, nb * 32, hd)[:, :, :cap], v.view(slots, kv, nb * 32, hd)[:, :, :cap]


def ranges(rows, past=0, starts=None, prefix=None, causal=True, window=0, shared=0):
    """first, lo, hi, pos of each row, one row at a time."""
    out = []
    for r in range(rows):
        i, n = past + r, past + rows
        if starts is None:
            d, s, e = 0, 0, n
        else:
            d = max([x for x in range(len(starts)) if starts[x] <= r], default=-1)
            if d < 0 or d >= len(starts) - 1:
                out.append((0, 0, 0, 0))
                continue
            s, e = past + starts[d], min(past + starts[d + 1], n)
        lo, hi = s, (i + 1 if causal else e)
        if window:
            lo = max(lo, i - window + 1)
            hi = hi if causal else min(hi, i + window)
        if prefix is not None:
            hi = max(hi, min(s + prefix[d], e))
        out.append((min(shared, i + 1 if causal else n), lo, hi, i - s))
    return torch.tensor(out, dtype=torch.int32).reshape(rows, 4).T.contiguous()


def visible(table, keys):
    j = torch.arange(keys)[None]
    f, lo, hi = (t[:, None] for t in table[:3].long())
    return (j < f) | ((j >= lo) & (j < hi))


def attend(q, k, v, seen, at, scale, softcap=0.0, slopes=None, decode=False):
    """(context, allowed error) in f64. q [rows, heads, hd]; k, v [kv, keys, hd]; seen [rows, keys]; at [rows]
    the rows' own positions. Keys that no row sees may hold anything."""
    rows, heads, hd = q.shape
    kv, keys, _ = k.shape
    out = torch.zeros(rows, heads, hd, dtype=torch.float64)
    tol = torch.zeros_like(out)
    dist = (at.double()[:, None] - torch.arange(keys)[None]).abs()
    live = seen.any(0)
    for h in range(heads):
        kh = torch.where(live[:, None], k[h // (heads // kv)].double(), 0.0)
        vh = torch.where(live[:, None], v[h // (heads // kv)].double(), 0.0)
        qh = q[:, h].double()
        s = qh @ kh.T * scale
        mag = qh.abs() @ kh.abs().T * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        b = float(slopes[h]) * dist if slopes is not None else torch.zeros_like(dist)
        s = s - b
        d = U * (hd + 8) * mag + 16 * U * softcap + 8 * U * (s.abs() + b)
        if decode:
            d = d + 2.0 ** -22 * mag + 2.0 ** -25 * scale * kh.abs().sum(-1)[None]
        s = torch.where(seen, s, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        n = seen.sum(-1, keepdim=True).double()
        total = p.sum(-1, keepdim=True).clamp(min=1e-300)
        p = p / total
        y = p @ vh
        d = torch.where(seen, d, 0.0)
        w = 2.0 ** -22 if decode else H
        off = (p * (w + d + 2 * n * U)) @ vh.abs() + 2.0 ** -25 * (seen / total) @ vh.abs()
        off = off + y.abs() * ((p * d).sum(-1, keepdim=True) + 2 * n * U + 4 * U)
        if not decode:
            off = off + y.abs() * (H + 2.0 ** -25 * n / total)
        off = 1.02 * off + y.abs() * (U if decode else H) + (0.0 if decode else 2.0 ** -25)
        out[:, h], tol[:, h] = y, off
    return out, tol


def rotate(x, pos, rot, theta, div=None, mscale=1.0, interleaved=False):
    """x [rows, heads, hd] in f64, rotated pair by pair."""
    y = x.double().clone()
    for d in range(rot // 2):
        a = pos.double() * theta ** (-2.0 * d / rot) / (1.0 if div is None else float(div[d]))
        i, j = (2 * d, 2 * d + 1) if interleaved else (d, d + rot // 2)
        c, s = (mscale * torch.cos(a))[:, None], (mscale * torch.sin(a))[:, None]
        y[..., i], y[..., j] = x[..., i].double() * c - x[..., j].double() * s, x[..., i].double() * s + x[..., j].double() * c
    return y
