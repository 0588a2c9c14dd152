"""Inputs, f64 results and error bounds for attention over packed sequences."""

from __future__ import annotations

import itertools

import numpy as np
import torch

import window_cases


def inputs(lengths, h, hk, d, dtype, *, before=0, behind=0, seed=0, junk=0.0):
    """offsets, and q, k, v, dy [tokens, heads, d], with `junk` in the rows of no sequence."""
    at = [before, *(before + n for n in itertools.accumulate(lengths))]
    t = at[-1] + behind
    g = torch.Generator().manual_seed(seed)
    x = [torch.randn(t, n, d, generator=g).to(dtype) for n in (h, hk, hk, h)]
    for y in x:
        y[:before] = junk
        y[at[-1]:] = junk
    return at, x


def expected(at, q, k, v, dy, window=0, scale=None):
    """{name: (f64 value, bound)} as window_cases.expected, sequence by sequence."""
    out = {}
    for name, like in (("out", q), ("dq", q), ("dk", k), ("dv", v)):
        out[name] = (np.zeros(like.shape), np.zeros(like.shape))
    for a, b in itertools.pairwise(at):
        if a == b:
            continue
        part = [x[a:b].transpose(0, 1)[None] for x in (q, k, v, dy)]
        for name, (value, bound) in window_cases.expected(*part, min(window, b - a) or b - a, 0, scale).items():
            out[name][0][a:b] = value[0].swapaxes(0, 1)
            out[name][1][a:b] = bound[0].swapaxes(0, 1)
    return out
