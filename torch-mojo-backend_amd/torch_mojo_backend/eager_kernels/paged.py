"""Calls of the paged key/value cache's kernels (csrc/paged_cache.hip,
csrc/paged_attention.hip) on mojo tensors.

Arguments are checked by their metadata in `torch_mojo_backend.ops`; what the
device alone knows (positions, page numbers) the kernels check, and an entry
out of range raises IndexError at the next device-to-host read, like an
embedding index.  As everywhere in this package outputs and workspaces are
allocated here and launches go to the null stream, that of the tensors' device.
"""

from __future__ import annotations

import contextlib

import torch

from . import PagedCache, check, materialize_touched
from . import native_lib as lib
from .aten_fast import _PAGE_ERROR, _STREAM, _alloc, _code, _error_slot, _workspace, alloc_bthd, materialize_contiguous
from ..mojo_device import torch_mojo_tensor as _tensor_mod

MT = _tensor_mod.TorchMojoTensor


def describe(cache) -> PagedCache:
    """The kernels' description of a cache's pages."""
    k, v, ks, vs = cache.k, cache.v, cache.k_scales, cache.v_scales
    d = PagedCache()
    d.k, d.v = k._ptr, v._ptr
    d.k_phs[:], d.v_phs[:] = k._strides[:3], v._strides[:3]
    if ks is not None:
        d.k_scales, d.v_scales = ks._ptr, vs._ptr
        d.ks_phs[:], d.vs_phs[:] = ks._strides[:3], vs._strides[:3]
    d.num_pages, d.page_size, d.kv_heads, d.d = cache.num_pages, cache.page_size, cache.kv_heads, cache.head_dim
    d.dtype, d.bits = _code(k._dtype), 4 if ks is not None else 0
    return d


def _on(device: int):
    """A context in which `device` is current: a launch on the null stream
    goes to the current device."""
    if _tensor_mod.storage_kind() == "cuda" and torch.cuda.current_device() != device:
        return torch.cuda.device(device)
    return contextlib.nullcontext()


def _rows(t: MT) -> MT:
    """t itself when its rows can be read 16 bytes at a time, else a copy."""
    if t._strides[3] == 1 and t._ptr % 16 == 0 and all(st * t._itemsize % 16 == 0 for st in t._strides[:3]):
        return t
    return materialize_contiguous(t)


def _bht(t: MT):
    return t._strides[:3]


def _seqs(table: MT, starts: MT, counts):
    return table._ptr, table._strides[0], table._shape[1], starts._ptr, counts._ptr if counts is not None else None


def append(cache, table, starts, k, v, cos, sin, q, counts):
    b, _, t, d = k._shape
    written = (cache.k, cache.v) if cache.k_scales is None else (cache.k, cache.v, cache.k_scales, cache.v_scales)
    materialize_touched((*written, table, starts, k, v, cos, sin, q, counts), None, True)
    dev = k._device
    with _on(dev):
        k, v = _rows(k), _rows(v)
        out = None
        if q is not None:
            q = _rows(q)
            out = alloc_bthd(b, q._shape[1], t, d, q._dtype, dev)
        if cos is not None:
            cos, sin = (x if x._is_contiguous and x._ptr % 16 == 0 else materialize_contiguous(x) for x in (cos, sin))
        check(
            "mi355x_paged_append",
            lib().mi355x_paged_append(
                cache._desc, *_seqs(table, starts, counts), k._ptr, _bht(k), v._ptr, _bht(v),
                out._ptr if q is not None else None, _bht(out) if q is not None else None,
                q._ptr if q is not None else None, _bht(q) if q is not None else None,
                cos._ptr if cos is not None else None, sin._ptr if cos is not None else None,
                _code(cos._dtype) if cos is not None else 0, cos._shape[0] if cos is not None else 0,
                b, q._shape[1] if q is not None else 0, t, _code(k._dtype), _error_slot(dev, _PAGE_ERROR), _STREAM,
            ),
        )
    torch.autograd.graph.increment_version(written)
    return out


def gather(cache, table, starts, length, counts, dtype):
    b, dev = table._shape[0], table._device
    materialize_touched((cache.k, cache.v, cache.k_scales, cache.v_scales, table, starts, counts), None, False)
    with _on(dev):
        k, v = (alloc_bthd(b, cache.kv_heads, length, cache.head_dim, dtype, dev) for _ in range(2))
        check(
            "mi355x_paged_gather",
            lib().mi355x_paged_gather(k._ptr, _bht(k), v._ptr, _bht(v), cache._desc, *_seqs(table, starts, counts),
                                      b, length, _code(dtype), _error_slot(dev, _PAGE_ERROR), _STREAM),
        )
    return k, v


def attention(q, cache, table, starts, counts, window, sinks, scale):
    b, h, t, d = q._shape
    dev, code = q._device, _code(q._dtype)
    materialize_touched((q, cache.k, cache.v, cache.k_scales, cache.v_scales, table, starts, counts), None, False)
    with _on(dev):
        q = _rows(q)
        out = alloc_bthd(b, h, t, d, q._dtype, dev)
        ws = lib().mi355x_paged_attn_workspace_bytes(cache._desc, table._shape[1], b, h, t, window, sinks, code)
        hold, wptr = _workspace(ws, dev)
        check(
            "mi355x_paged_attn",
            lib().mi355x_paged_attn(out._ptr, _bht(out), q._ptr, _bht(q), cache._desc, *_seqs(table, starts, counts),
                                    b, h, t, scale, window, sinks, code, wptr, ws, _error_slot(dev, _PAGE_ERROR),
                                    _STREAM),
        )
    return out
