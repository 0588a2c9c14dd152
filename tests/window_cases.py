"""Inputs, f64 results and error bounds for sliding-window attention with sinks."""

from __future__ import annotations

import numpy as np
import torch

from oracle import paged as oracle
from paged_cases import STEP, np64


def inputs(b, h, hk, t, d, dtype, seed=0):
    """q, k, v, dy [batch, heads, tokens, d] as views of [batch, tokens, heads, d]."""
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(b, t, n, d, generator=g).to(dtype).transpose(1, 2) for n in (h, hk, hk, h)]


def expected(q, k, v, dy, window, sinks, scale=None):
    """{name: (f64 value, bound)}.  With u half a step of the type: the
    weights are rounded to it (in sums and quotient: twice), so are dS and the
    saved o, whose error reaches D = dy.o, and each result; f32 sums of n
    products add n + 8 steps of 2^-24 of the absolute sum.  Below f16's least
    normal number, 2^-14, half a step is 2^-25 and no share of the value: `sub`
    for each rounding of a weight, of dS and of a result."""
    u, dtype = STEP[q.dtype], q.dtype
    qn, kn, vn, dn = (np64(x) for x in (q, k, v, dy))
    b, h, t, d = qn.shape
    hk, g = kn.shape[1], h // kn.shape[1]
    sc = d ** -0.5 if scale is None else scale
    kk, vv = np.repeat(kn, g, 1), np.repeat(vn, g, 1)
    o, lse = oracle.window_forward(qn, kn, vn, window, sinks, scale)
    dq, dk, dv = oracle.window_backward(dn, qn, kn, vn, window, sinks, scale)
    mask = oracle.window_mask(t, window, sinks)
    s = np.where(mask, sc * (qn @ kk.swapaxes(-1, -2)), -np.inf)
    p = np.exp(s - lse[..., None])
    fold = lambda x: x.reshape(b, hk, g, t, d).sum(2)  # noqa: E731
    tiny = 2.0 ** -24
    w = u if dtype != torch.float32 else 0.0
    sub = 2.0 ** -25 if dtype == torch.float16 else 0.0
    # relative error of a weight: rounding, and what the score's f32 sum and exp move
    dscore = (d + 16) * tiny * (abs(sc) * (np.abs(qn) @ np.abs(kk).swapaxes(-1, -2)) * mask).max() + 16 * tiny
    pe = w + 2 * dscore + (t + 8) * tiny
    o_err = 2 * pe * (p @ np.abs(vv)) + u * np.abs(o) + sub * (1 + 2 * (mask @ np.abs(vv)))
    dp = dn @ vv.swapaxes(-1, -2)
    delta = (dn * o).sum(-1, keepdims=True)
    delta_err = (np.abs(dn) * o_err).sum(-1, keepdims=True) + (d + 8) * tiny * (np.abs(dn) * np.abs(o)).sum(-1, keepdims=True)
    dp_err = (d + 8) * tiny * (np.abs(dn) @ np.abs(vv).swapaxes(-1, -2))
    ds = p * (dp - delta)
    ds_err = (pe + w) * np.abs(ds) + p * (delta_err + dp_err) + sub * mask
    n = (t * g + 8) * tiny  # sums over keys or over queries and heads
    at = lambda x: x.swapaxes(-1, -2)  # noqa: E731
    dq_err = abs(sc) * ((ds_err + n * np.abs(ds)) @ np.abs(kk)) + 2 * u * np.abs(dq) + sub
    dk_err = fold(abs(sc) * (at(ds_err + n * np.abs(ds)) @ np.abs(qn))) + 2 * u * np.abs(dk) + sub
    dv_err = fold((at((pe + n) * p + sub * mask)) @ np.abs(dn)) + u * np.abs(dv) + sub
    return {"out": (o, o_err), "dq": (dq, dq_err), "dk": (dk, dk_err), "dv": (dv, dv_err)}
