"""Calls of the kernels of packed sequences (csrc/packed_plan.hip,
csrc/attention_packed.hip) on mojo tensors.

Arguments are checked in `torch_mojo_backend.packing` and
`torch_mojo_backend.ops`; the offsets, which the device alone knows, the kernels
check, and raise at the next device-to-host read.  Outputs and workspaces are
allocated here; launches go to the null stream of the tensors' device.
"""

from __future__ import annotations

import math

import torch

from . import check, lazy_live, materialize_touched
from . import native_lib as lib
from .aten_fast import (
    _PACKING_ERROR, _STREAM, _alloc, _code, _contig, _error_slot, _mark_cat_ready, _workspace, materialize_contiguous,
)
from .paged import on_device
from ..mojo_device.torch_mojo_tensor import TorchMojoTensor as MT

_MOST_ROW_BYTES = 2 ** 26 - 64
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def plan(offsets: MT, tokens: int):
    """(plan, positions) of a batch."""
    if lazy_live():
        materialize_touched((offsets,), None, False)
    return on_device(offsets._device, _plan, offsets, tokens, offsets._device)


def _plan(offsets, tokens, dev):
    offsets = _contig(offsets)
    n = offsets._shape[0] - 1
    size = lib().mi355x_packed_plan_bytes(n, tokens)
    out, positions = _alloc((size,), torch.uint8, dev), _alloc((tokens,), torch.int32, dev)
    check(
        "mi355x_packed_plan",
        lib().mi355x_packed_plan(out._ptr, size, positions._ptr, offsets._ptr, n, tokens,
                                 _error_slot(dev, _PACKING_ERROR), _STREAM),
    )
    return out, positions


def _rows(t: MT) -> MT:
    """t itself when its rows can be read 16 bytes at a time and lie less than
    64 MB apart (the kernels' offsets in a tile of 64 have 32 bits), else a copy."""
    st, n = t._strides, t._itemsize
    if st[2] == 1 and not (t._ptr | st[0] * n | st[1] * n) & 15 and st[0] * n <= _MOST_ROW_BYTES:
        return t
    return materialize_contiguous(t)


def _th(t: MT):
    return t._strides[:2]


def ready(q, k, v, sequences) -> bool:
    """Whether a call needs no further look (the checks of
    torch_mojo_backend.ops, which name what is wrong, take as long as a small
    call's kernel)."""
    if type(q) is not MT or type(k) is not MT or type(v) is not MT or not getattr(sequences, "on_mojo", False):
        return False
    qs, ks, dev, dtype = q._shape, k._shape, q._device, q._dtype
    return (len(qs) == len(ks) == 3 and ks == v._shape and qs[0] == ks[0] == sequences.tokens and qs[2] == ks[2]
            and qs[0] and ks[1] and qs[1] and qs[1] % ks[1] == 0 and 0 < qs[2] <= 256 and qs[2] % 8 == 0
            and dtype in _FLOATS and dtype is k._dtype is v._dtype and dev == k._device == v._device == sequences._plan._device)


def attention(q, k, v, sequences, window, scale):
    """Without a graph; the gradient's form is mojo_device_autograd's _PackedAttention."""
    if lazy_live():
        materialize_touched((q, k, v), None, False)
    return on_device(q._device, attention_forward, q, k, v, sequences, window, scale)[0]


def attention_forward(q: MT, k: MT, v: MT, sequences, window, scale, keep_low=False):
    """(out [tokens, heads, head_dim], lse f32 [heads, tokens], low): low is
    what rounding took from a 16-bit out, for the backward's row terms."""
    q, k, v = _rows(q), _rows(k), _rows(v)
    t, h, d = q._shape
    out = _alloc((t, h, d), q._dtype, q._device)
    lse = _alloc((h, t), torch.float32, q._device)
    low = _alloc((t, h, d), q._dtype, q._device) if keep_low and q._dtype is not torch.float32 else None
    check(
        "mi355x_packed_attn_fwd",
        lib().mi355x_packed_attn_fwd(out._ptr, _th(out), low._ptr if low is not None else None, lse._ptr, q._ptr, _th(q),
                                     k._ptr, _th(k), v._ptr, _th(v), sequences._plan._ptr, sequences.count, t, h,
                                     k._shape[1], d, _scale(scale, d), window, _code(q._dtype), _STREAM),
    )
    return out, lse, low


def attention_backward(grad: MT, q: MT, k: MT, v: MT, out: MT, lse: MT, low, sequences, window, scale):
    """(dq, dk, dv): dense, or the parts of one dense tensor."""
    if grad._dtype != q._dtype:
        grad = materialize_contiguous(grad, q._dtype)
    # (a leaf's gradient is kept, and must not share memory with a cat of it)
    together = q._holder is k._holder is v._holder and not (q.is_leaf or k.is_leaf or v.is_leaf)
    grad, q, k, v = _rows(grad), _rows(q), _rows(k), _rows(v)
    # (as the forward made them, unless a saved-tensor hook gave back other ones)
    out, lse, low = _contig(out), _contig(lse), _contig(low) if low is not None else None
    t, h, d = q._shape
    hk, code, library = k._shape[1], _code(q._dtype), lib()
    if together and hk == h:
        # slices of one projection: side by side, so that the backward of its
        # split is a view (aten_fast._mark_cat_ready)
        rows = _alloc((t, 3, h, d), q._dtype, q._device)
        dq, dk, dv = (MT._view_of(rows, (t, h, d), (3 * h * d, d, 1), i * h * d) for i in range(3))
        _mark_cat_ready(rows)
    else:
        dq, dk, dv = (_alloc(x._shape, q._dtype, q._device) for x in (q, k, v))
    if hk < h and q._dtype is not torch.float32:
        ws = library.mi355x_packed_attn_bwd_workspace_bytes_for(sequences.count, t, h, hk, d, code)
    else:  # (the most of any type)
        ws = library.mi355x_packed_attn_bwd_workspace_bytes(sequences.count, t, h, hk, d)
    hold, wptr = _workspace(ws, q._device)
    check(
        "mi355x_packed_attn_bwd",
        library.mi355x_packed_attn_bwd(
            dq._ptr, _th(dq), dk._ptr, _th(dk), dv._ptr, _th(dv), grad._ptr, _th(grad), q._ptr, _th(q), k._ptr, _th(k),
            v._ptr, _th(v), out._ptr, _th(out), low._ptr if low is not None else None, lse._ptr, sequences._plan._ptr,
            sequences.count, t, h, hk, d, _scale(scale, d), window, code, wptr, ws, _STREAM,
        ),
    )
    return dq, dk, dv


def _scale(scale, d) -> float:
    return 1.0 / math.sqrt(d) if scale is None else scale
