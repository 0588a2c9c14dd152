"""f64 results and error bounds of rotary positions and token log-probabilities."""

from __future__ import annotations

import numpy as np
import torch

from paged_cases import STEP, np64


def turned(x, positions, frequencies, interleaved, scale, inverse=False):
    """(value, bound) of rows x [batch, heads, tokens, d].  The rest of a turn is
    rounded to f32 (half a step below 1/2: 2^-26 of a turn) from a product in f64
    (two roundings of its turns); sine and cosine are good to 2^-22 with the
    scale's product, and the two products and their sum add 3 roundings."""
    v, n = np64(x), 2 * len(frequencies)
    pos = np.broadcast_to(np64(positions), (v.shape[0], v.shape[2]))
    angle = pos[:, None, :, None] * np64(frequencies)
    j = np.arange(n // 2)
    a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + n // 2)
    cos, sin = scale * np.cos(angle), scale * np.sin(angle) * (-1 if inverse else 1)
    out, bound = v.copy(), np.zeros_like(v)
    out[..., a], out[..., b] = v[..., a] * cos - v[..., b] * sin, v[..., b] * cos + v[..., a] * sin
    off = 2 * np.pi * (2.0 ** -26 + np.abs(angle) / (2 * np.pi) * 2.0 ** -51) + 2.0 ** -22 + 3 * 2.0 ** -24
    size = abs(scale) * (np.abs(v[..., a]) + np.abs(v[..., b])) * off
    sub = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    for c in (a, b):
        bound[..., c] = size + STEP[x.dtype] * np.abs(out[..., c]) + sub
    return out, bound


def logits(n, c, dtype, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (spread * torch.randn(n, c, generator=g)).to(dtype)
    return x, torch.randint(0, c, (n,), generator=g)


def best_of(x, top):
    """Tokens of the largest entries: NaN first, then by value, then by index."""
    v = np64(x)
    v = np.where(np.isnan(v), np.inf, v) if np.isnan(v).any() else v
    order = np.lexsort((np.broadcast_to(np.arange(v.shape[1]), v.shape), -v, ~np.isnan(np64(x))), axis=-1)
    return order[:, :top]


def expected(x, tokens, top=0, grads=(None, None, None), ignore_index=-100):
    """{name: (value, bound)}.  A term exp(x - m) is off by 2^-22 and by the
    rounding of its exponent, |x - m| 2^-23; a lane adds 128 of them and the sums
    go through a tree and up to 16 segments a thread: 160 roundings.  The logarithm
    is good to 2^-22 of its value."""
    v = np64(x)
    n, c = v.shape
    m = v.max(-1, keepdims=True)
    z = v - m
    e = np.exp(z)
    s = e.sum(-1, keepdims=True)
    p, ls = e / s, np.log(s)
    logp = z - ls
    near = np.where(p > 0, z, 0.0)  # -inf adds nothing
    t, t2 = (p * near).sum(-1, keepdims=True), (p * near * near).sum(-1, keepdims=True)
    h = ls - t
    sums = 160 * 2.0 ** -24 + 2.0 ** -22
    e_s = sums + np.abs(t) * 2.0 ** -23
    ls_err = e_s + 2.0 ** -22 * np.abs(ls)
    h_err = ls_err + (sums + e_s) * np.abs(t) + t2 * 2.0 ** -23 + 2.0 ** -22 * (np.abs(ls) + np.abs(t))
    rows = np.arange(n)
    out = {}

    def at(cols):  # log-probabilities of columns [n, k]
        value, zz = np.take_along_axis(logp, cols, 1), np.take_along_axis(z, cols, 1)
        size = np.where(np.isfinite(zz), np.abs(zz), 0.0)
        return value, ls_err + 2.0 ** -23 * (size + np.abs(ls)) + 2.0 ** -24 * np.where(np.isfinite(value), np.abs(value), 0.0)

    given = None
    if tokens is not None:
        tk = tokens.numpy()
        given = tk != ignore_index
        value, bound = at(np.where(given, tk, 0)[:, None])
        out["logprobs"] = (np.where(given, value[:, 0], 0.0), np.where(given, bound[:, 0], 0.0))
    out["entropy"] = (h[:, 0], h_err[:, 0])
    order = best_of(x, top) if top else None
    if top:
        out["top_logprobs"] = at(order)
        out["top_tokens"] = order
    if any(g is not None for g in grads):
        g = np.zeros((n, c))
        size = np.zeros((n, 1))
        if grads[0] is not None:
            d = np64(grads[0]) * given
            g[rows, np.where(given, tk, 0)] += d
            size += np.abs(d)[:, None]
        if grads[2] is not None:
            np.add.at(g, (rows[:, None], order), np64(grads[2]))
            size += np.abs(np64(grads[2])).sum(-1, keepdims=True)
        ones = np.abs(g)
        gh = np64(grads[1])[:, None] if grads[1] is not None else np.zeros((n, 1))
        lp = np.where(p > 0, logp, 0.0)
        dx = g - p * (g.sum(-1, keepdims=True) + gh * (lp + h))
        rel = (np.abs(near) + np.abs(ls)) * 2.0 ** -22 + e_s + 2.0 ** -21
        part = size + np.abs(gh) * (np.abs(lp) + np.abs(h))
        bound = p * (rel * part + np.abs(gh) * (np.abs(lp) * 2.0 ** -21 + h_err) + (top + 4) * 2.0 ** -24 * part)
        bound += 4 * 2.0 ** -24 * (ones + np.abs(dx)) + STEP[x.dtype] * np.abs(dx) + 2.0 ** -120 * part
        if x.dtype == torch.float16:
            bound += 2.0 ** -25
        out["dx"] = (dx, bound)
    return out
