"""Calls of the paged key/value cache's kernels (csrc/paged_cache.hip,
csrc/paged_attention.hip) on mojo tensors.

Arguments are checked by their metadata in `torch_mojo_backend.ops`; what the
device alone knows (positions, page numbers) the kernels check, and an entry
out of range raises IndexError at the next device-to-host read, like an
embedding index.  As everywhere in this package outputs and workspaces are
allocated here and launches go to the null stream, that of the tensors' device.
"""

from __future__ import annotations

import torch

from . import PagedCache, check, lazy_live, materialize_touched
from . import native_lib as lib
from .aten_fast import _PAGE_ERROR, _STREAM, _code, _error_slot, _workspace, alloc_bthd, materialize_contiguous
from ..mojo_device import torch_mojo_tensor as _tensor_mod

MT = _tensor_mod.TorchMojoTensor
_INT32 = torch.int32
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


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


# ---------------------------------------------------------------------------
# Whether a call is one that needs no further look: a decode step is a few
# microseconds of kernel, and the checks of torch_mojo_backend.ops, which name
# what is wrong, take longer than that.
# ---------------------------------------------------------------------------
def seqs_ok(cache, table, starts, counts) -> bool:
    if not cache.on_mojo or type(table) is not MT or type(starts) is not MT:
        return False
    dev, shape = cache.k._device, table._shape
    if not (table._dtype is _INT32 and starts._dtype is _INT32 and len(shape) == 2 and shape[1] and table._strides[1] == 1
            and table._device == dev and starts._device == dev and starts._shape == shape[:1]
            and starts._strides == (1,)):
        return False
    return counts is None or (type(counts) is MT and counts._dtype is _INT32 and counts._shape == shape[:1]
                              and counts._strides == (1,) and counts._device == dev)


def rows_ok(cache, t, batch, like=None) -> bool:
    """[batch, any heads, any tokens, head_dim] of the pages' type, or for 4-bit
    pages of a float type, that of `like` where given."""
    if type(t) is not MT or t.requires_grad:
        return False
    shape, dtype = t._shape, t._dtype
    return (len(shape) == 4 and shape[0] == batch and shape[3] == cache.head_dim and t._device == cache.k._device
            and (dtype is cache.dtype if cache.bits != 4 else dtype in _FLOATS if like is None else dtype is like._dtype))


def on_device(device: int, call, *args):
    """call(*args) with `device` current: a launch on the null stream goes to
    the current device."""
    if _tensor_mod.storage_kind() == "cuda" and torch._C._cuda_getDevice() != device:
        with torch.cuda.device(device):
            return call(*args)
    return call(*args)


def _rows(t: MT, written=()) -> MT:
    """t itself when its rows can be read 16 bytes at a time and do not lie in
    a storage that the call writes (moved tokens: views of the pages), else a
    copy."""
    st, n = t._strides, t._itemsize
    if st[3] == 1 and not (t._ptr | st[0] * n | st[1] * n | st[2] * n) & 15 and id(t._holder) not in written:
        return t
    return materialize_contiguous(t)


def _bht(t: MT):
    return t._strides[:3]


def _seqs(table: MT, starts: MT, counts):
    return table._ptr, table._strides[0], table._shape[1], starts._ptr, counts._ptr if counts is not None else None


def append(cache, table, starts, k, v, cos, sin, q, counts):
    if lazy_live():
        materialize_touched((*cache.tensors, table, starts, k, v, cos, sin, q, counts), None, True)
    dev = k._device
    out = on_device(dev, _append, cache, table, starts, k, v, cos, sin, q, counts, dev)
    torch._C._increment_version(cache.tensors)
    return out


def _append(cache, table, starts, k, v, cos, sin, q, counts, dev):
    b, _, t, d = k._shape
    k, v = _rows(k, cache.holders), _rows(v, cache.holders)
    out, q_args, rope = None, (None, None, None, None), (None, None, 0, 0)
    heads = 0
    if q is not None:
        q, heads = _rows(q, cache.holders), q._shape[1]
        out = alloc_bthd(b, heads, t, d, q._dtype, dev)
        q_args = out._ptr, _bht(out), q._ptr, _bht(q)
    if cos is not None:
        cos, sin = (x if x._is_contiguous and x._ptr % 16 == 0 else materialize_contiguous(x) for x in (cos, sin))
        rope = cos._ptr, sin._ptr, _code(cos._dtype), cos._shape[0]
    check(
        "mi355x_paged_append",
        lib().mi355x_paged_append(cache._desc, *_seqs(table, starts, counts), k._ptr, _bht(k), v._ptr, _bht(v), *q_args,
                                  *rope, b, heads, t, _code(k._dtype), _error_slot(dev, _PAGE_ERROR), _STREAM),
    )
    return out


def gather(cache, table, starts, length, counts, dtype):
    if lazy_live():
        materialize_touched((*cache.tensors, table, starts, counts), None, False)
    return on_device(table._device, _gather, cache, table, starts, length, counts, dtype, table._device)


def _gather(cache, table, starts, length, counts, dtype, dev):
    b = table._shape[0]
    k, v = (alloc_bthd(b, cache.kv_heads, length, cache.head_dim, dtype, dev) for _ in range(2))
    check(
        "mi355x_paged_gather",
        lib().mi355x_paged_gather(k._ptr, _bht(k), v._ptr, _bht(v), cache._desc, *_seqs(table, starts, counts),
                                  b, length, _code(dtype), _error_slot(dev, _PAGE_ERROR), _STREAM),
    )
    return k, v


def attention(q, cache, table, starts, counts, window, sinks, scale):
    if lazy_live():
        materialize_touched((q, *cache.tensors, table, starts, counts), None, False)
    return on_device(q._device, _attention, q, cache, table, starts, counts, window, sinks, scale, q._device)


def _attention(q, cache, table, starts, counts, window, sinks, scale, dev):
    b, h, t, d = q._shape
    q = _rows(q)
    code = _code(q._dtype)
    out = alloc_bthd(b, h, t, d, q._dtype, dev)
    library = lib()
    ws = library.mi355x_paged_attn_workspace_bytes(cache._desc, table._shape[1], b, h, t, window, sinks, code)
    hold, wptr = _workspace(ws, dev)
    check(
        "mi355x_paged_attn",
        library.mi355x_paged_attn(out._ptr, _bht(out), q._ptr, _bht(q), cache._desc, *_seqs(table, starts, counts),
                                  b, h, t, scale, window, sinks, code, wptr, ws, _error_slot(dev, _PAGE_ERROR), _STREAM),
    )
    return out
