"""Paged key/value cache and sliding-window attention with sinks, from their
definitions in f64 (the reference has no counterpart; pinned in
tests/test_paged.py against closed forms and brute force)."""

from __future__ import annotations

import math

import numpy as np

GROUP = 32


def turn(x, cos, sin):
    """x [..., d] * cos + rotate_half(x) * sin."""
    x, cos, sin = (np.asarray(v, dtype=np.float64) for v in (x, cos, sin))
    half = x.shape[-1] // 2
    return x * cos + np.concatenate([-x[..., half:], x[..., :half]], axis=-1) * sin


def quantize(x):
    """x [..., d] as (codes, scale, minimum): one code a channel, one scale and
    minimum (f16) a group of 32."""
    x = np.asarray(x, dtype=np.float64)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    bad = ~np.isfinite(g).all(-1)
    g = np.clip(np.where(np.isfinite(g), g, 0.0), -61440.0, 61440.0)
    low = g.min(-1)
    scale = ((g.max(-1) - low) / 15.0).astype(np.float32).astype(np.float16)
    low = low.astype(np.float32).astype(np.float16)
    scale[bad] = low[bad] = np.nan
    s, m = scale.astype(np.float64)[..., None], low.astype(np.float64)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        codes = np.where(s > 0, np.clip(np.rint((g - m) / s), 0, 15), 0.0)
    return codes.reshape(x.shape).astype(np.int64), scale, low


def values(codes, scale, low):
    """The f64 values that codes stand for."""
    c = codes.reshape(*codes.shape[:-1], codes.shape[-1] // GROUP, GROUP)
    return (low.astype(np.float64)[..., None] + scale.astype(np.float64)[..., None] * c).reshape(codes.shape)


def place_of(channel, d):
    """(byte, nibble) of a channel in a row of d / 2 bytes."""
    s, g, e = channel // 32, channel % 32 // 8, channel % 8
    n = e // 2 + 4 * (e % 2)
    return 4 * (g * (d // 32) + s) + n // 2, n % 2


def visible(p, j, window, sinks):
    return j <= p and (window <= 0 or p - j < window or j < sinks)


def attend(q, k, v, positions, window=0, sinks=0, scale=None):
    """o [H, T, d] of queries q [H, T, d] at `positions` over rows k, v [Hk, n,
    d]; a query at a negative position, or one that sees nothing, gives zero."""
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    h, t, d = q.shape
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    g = h // k.shape[0]
    j = np.arange(k.shape[1])
    out = np.zeros_like(q)
    for i, p in enumerate(positions):
        keep = (j <= p) & ((j < sinks) | (p - j < window) if window > 0 else True)
        if p < 0 or not keep.any():
            continue
        for a in range(h):
            s = scale * (k[a // g][keep] @ q[a, i])
            w = np.exp(s - s.max())
            out[a, i] = (w / w.sum()) @ v[a // g][keep]
    return out


def window_mask(t, window, sinks=0):
    i, j = np.arange(t)[:, None], np.arange(t)[None, :]
    return (j <= i) & ((i - j < window) | (j < sinks))


def window_forward(q, k, v, window, sinks=0, scale=None):
    """(o, lse) of q [B, H, T, d] over k, v [B, Hk, T, d]."""
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    g = q.shape[1] // k.shape[1]
    k, v = np.repeat(k, g, 1), np.repeat(v, g, 1)
    s = np.where(window_mask(q.shape[2], window, sinks), scale * (q @ k.swapaxes(-1, -2)), -np.inf)
    m = s.max(-1, keepdims=True)
    lse = (m + np.log(np.exp(s - m).sum(-1, keepdims=True)))[..., 0]
    return np.exp(s - lse[..., None]) @ v, lse


def window_backward(do, q, k, v, window, sinks=0, scale=None):
    """(dq, dk, dv); dk and dv of a K/V head sum over its query heads."""
    do, q, k, v = (np.asarray(x, dtype=np.float64) for x in (do, q, k, v))
    b, h, t, d = q.shape
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    hk, g = k.shape[1], h // k.shape[1]
    o, lse = window_forward(q, k, v, window, sinks, scale)
    kk, vv = np.repeat(k, g, 1), np.repeat(v, g, 1)
    s = np.where(window_mask(t, window, sinks), scale * (q @ kk.swapaxes(-1, -2)), -np.inf)
    p = np.exp(s - lse[..., None])
    ds = p * (do @ vv.swapaxes(-1, -2) - (do * o).sum(-1, keepdims=True))
    fold = lambda x: x.reshape(b, hk, g, t, d).sum(2)  # noqa: E731
    return (scale * ds @ kk, fold(scale * ds.swapaxes(-1, -2) @ q), fold(p.swapaxes(-1, -2) @ do))
