"""Calls of the rotary positions' and the token log-probabilities' kernels
(csrc/rope_at.hip, csrc/logprobs.hip) on mojo tensors.

Arguments are checked in `torch_mojo_backend.ops`.  Outputs and workspaces are
allocated here; launches go to the null stream of the tensors' device.
"""

from __future__ import annotations

import torch

from . import check
from . import native_lib as lib
from .aten_fast import (
    _STREAM, _TARGET_ERROR, _alloc, _code, _contig, _error_slot, _workspace, alloc_bthd, materialize_contiguous,
)
from ..mojo_device.torch_mojo_tensor import TorchMojoTensor as MT

_FLOATS, _INTS = (torch.bfloat16, torch.float16, torch.float32), (torch.int32, torch.int64)


def _bht(t: MT):
    """(batch, head, token) strides of [batch, heads, tokens, d] or [tokens, heads, d]."""
    st = t._strides
    return st[:3] if len(st) == 4 else (0, st[1], st[0])


def ready(q, k, positions, frequencies) -> bool:
    """Whether a rotary call needs no further look (as packed.ready)."""
    if type(q) is not MT or type(positions) is not MT or type(frequencies) is not MT or not (k is None or type(k) is MT):
        return False
    shape, dev, dtype, ps, fs = q._shape, q._device, q._dtype, positions._shape, frequencies._shape
    if len(shape) == 4:
        outer = (shape[0], shape[2])
    elif len(shape) == 3:
        outer = shape[:1]
    else:
        return False
    if k is not None:
        ks = k._shape
        if not (len(ks) == len(shape) and ks[0] == shape[0] and ks[2] == shape[2] and ks[-1] == shape[-1]
                and k._dtype is dtype and k._device == dev):
            return False
    return ((ps == outer or ps == outer[-1:]) and positions._dtype in _INTS and len(fs) == 1 and 2 * fs[0] <= shape[-1] <= 4096
            and frequencies._dtype is torch.float64 and dtype in _FLOATS and dev == positions._device == frequencies._device)


def _channels(t):
    """t itself when its channels lie side by side, else a copy."""
    return t if t is None or t._strides[-1] == 1 else materialize_contiguous(t)


def _side(t):
    """(out, its pointer and strides, t's pointer and strides, heads) for t, of
    channels side by side, or None."""
    if t is None:
        return None, (None, (0, 0, 0), None, (0, 0, 0), 0)
    out = alloc_bthd(*t._shape, t._dtype, t._device) if len(t._shape) == 4 else _alloc(t._shape, t._dtype, t._device)
    return out, (out._ptr, _bht(out), t._ptr, _bht(t), t._shape[1])


def rotary(q, k, positions: MT, frequencies: MT, interleaved, scale, inverse):
    """(q, k) turned; either may be None."""
    like = q if q is not None else k
    batch, seq = (like._shape[0], like._shape[2]) if len(like._shape) == 4 else (1, like._shape[0])
    if positions._strides and positions._strides[-1] != 1 and positions._shape[-1] > 1:
        positions = materialize_contiguous(positions)
    frequencies = _contig(frequencies)
    q, k = _channels(q), _channels(k)  # (copies are held until the launch)
    (qo, qa), (ko, ka) = _side(q), _side(k)
    check(
        "mi355x_rope_at",
        lib().mi355x_rope_at(*qa, *ka, positions._ptr, _code(positions._dtype),
                             positions._strides[0] if len(positions._shape) == 2 else 0, frequencies._ptr, batch, seq,
                             like._shape[-1], 2 * frequencies._shape[0], int(interleaved), scale, int(inverse),
                             _code(like._dtype), _STREAM),
    )
    return qo, ko


def logprobs_ready(x, tokens, top) -> bool:
    """Whether token_logprobs of rows needs no further look (as packed.ready)."""
    if type(x) is not MT or type(top) is not int or not (tokens is None or type(tokens) is MT):
        return False
    shape = x._shape
    return (len(shape) == 2 and 0 <= top <= 64 and 0 < shape[1] >= top and x._dtype in _FLOATS
            and (tokens is None or (tokens._dtype is torch.int64 and tokens._shape == shape[:1] and tokens._device == x._device)))


def logprobs_forward(x: MT, tokens, top, entropy, ignore_index, keep=False):
    """(logprobs, entropy, top_logprobs, top_tokens, stats) of x [n, vocab]; the
    rows' statistics where they are to be kept for the backward."""
    if x._strides[1] != 1 and x._shape[1] > 1 or x._strides[0] < 0:
        x = materialize_contiguous(x)
    (n, c), dev = x._shape, x._device
    code, library = _code(x._dtype), lib()
    f32 = torch.float32
    picked = _alloc((n,), f32, dev) if tokens is not None else None
    spread = _alloc((n,), f32, dev) if entropy else None
    best, order = (_alloc((n, top), f32, dev), _alloc((n, top), torch.int64, dev)) if top else (None, None)
    stats = _alloc((n, 2), f32, dev) if keep else None
    ws = library.mi355x_token_logprobs_workspace_bytes(n, c, top, code)
    hold, wptr = _workspace(ws, dev)
    error = _error_slot(dev, _TARGET_ERROR)  # (the first one allocates)
    tokens = _contig(tokens) if tokens is not None else None  # (a copy is held until the launch)
    at = lambda t: t._ptr if t is not None else None  # noqa: E731
    check(
        "mi355x_token_logprobs_fwd",
        library.mi355x_token_logprobs_fwd(at(picked), at(spread), at(stats), at(best), at(order), x._ptr, code,
                                          x._strides[0], at(tokens), n, c, top, ignore_index, error, wptr, ws, _STREAM),
    )
    return picked, spread, best, order, stats


def logprobs_backward(x: MT, tokens, stats, spread, order, d_picked, d_spread, d_best, ignore_index, dense_rows):
    """d_logits of x's dtype: dense, as a leaf's gradient is kept, or its rows
    padded to 8 elements, as the GEMMs behind a projection read them."""
    if x._strides[1] != 1 and x._shape[1] > 1 or x._strides[0] < 0:
        x = materialize_contiguous(x)
    (n, c), dev = x._shape, x._device
    ld = c if dense_rows else (c + 7) // 8 * 8
    dense = _alloc((n, ld), x._dtype, dev)
    dx = MT._view_of(dense, (n, c), (ld, 1), 0, ld == c)

    def grad(t):
        if t is None:
            return None
        return _contig(t) if t._dtype is torch.float32 else materialize_contiguous(t, torch.float32)

    d_picked, d_spread, d_best = grad(d_picked), grad(d_spread), grad(d_best)
    tokens, spread, order, stats = (t if t is None else _contig(t) for t in (tokens, spread, order, stats))
    at = lambda t: t._ptr if t is not None else None  # noqa: E731
    check(
        "mi355x_token_logprobs_bwd",
        lib().mi355x_token_logprobs_bwd(dx._ptr, ld, x._ptr, _code(x._dtype), x._strides[0], stats._ptr, at(spread),
                                        at(tokens), at(order), order._shape[1] if order is not None else 0,
                                        at(d_picked), at(d_spread), at(d_best), n, c, ignore_index, _STREAM),
    )
    return dx
