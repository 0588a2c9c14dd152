"""Fused ops of the Gemma-3-shaped workload: rotary embedding, GeGLU and
RMSNorm with a weight offset, attention over a sliding window with sinks; and
serving's: appending to a paged key/value cache and attention over it.

Torch has no single aten op for these (a model writes them as chains of
slice / neg / cat / mul / add, gelu + mul, and rms_norm with `1 + w`); the
functions here keep those semantics, run one gfx950 kernel each on the mojo
device, and fall back to the plain formula elsewhere (the CPU reference),
so a model written with them runs unchanged on both.  All but those of the
cache are differentiable.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from . import kv_cache
from .eager_kernels import aten_fast, materialize_touched, paged
from .masks import sliding_window_causal_mask
from .mojo_device.torch_mojo_tensor import TorchMojoTensor


def _on_mojo(*ts) -> bool:
    return all(isinstance(t, TorchMojoTensor) for t in ts)


def _needs_grad(*ts) -> bool:
    """Whether autograd records this call (otherwise the forward kernel is
    called directly, without an autograd Function's per-call cost)."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, cos, sin):
        ctx.save_for_backward(cos, sin)
        return aten_fast.rope_forward(x, cos, sin)

    @staticmethod
    def backward(ctx, grad):
        cos, sin = ctx.saved_tensors
        return aten_fast.rope_forward(grad, cos, sin, inverse=True), None, None


def rotary_embedding(x, cos, sin):
    """x * cos + rotate_half(x) * sin over the last dim of x [B, H, T, D], with
    rotate_half(x) = cat(-x[..., D/2:], x[..., :D/2]) and cos/sin [T, D]."""
    if (_on_mojo(x, cos, sin) and x.dim() == 4 and x.shape[-1] % 8 == 0
            and tuple(cos.shape) == (x.shape[2], x.shape[3]) and tuple(sin.shape) == tuple(cos.shape)
            and x.dtype in (torch.float32, torch.bfloat16, torch.float16)):
        if not _needs_grad(x, cos, sin):
            return aten_fast.rope_forward(x, cos, sin)
        return _Rope.apply(x, cos, sin)
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], dim=-1) * sin


class _GeGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up, approximate):
        ctx.save_for_backward(gate, up)
        ctx.approximate = approximate
        return aten_fast.geglu_forward(gate, up, approximate)

    @staticmethod
    def backward(ctx, grad):
        gate, up = ctx.saved_tensors
        if _on_mojo(grad) and grad.shape == gate.shape and grad.dtype == gate.dtype:
            with torch._C._AutoDispatchBelowAutograd():
                d_gate, d_up = aten_fast.geglu_backward(grad, gate, up, ctx.approximate)
            return d_gate, d_up, None
        act = F.gelu(gate, approximate=ctx.approximate)
        d_up = grad * act
        d_gate = torch.ops.aten.gelu_backward(grad * up, gate, approximate=ctx.approximate)
        return d_gate, d_up, None


def geglu(gate, up, approximate="tanh"):
    """gelu(gate) * up."""
    if (_on_mojo(gate, up) and gate.shape == up.shape and gate.dtype == up.dtype
            and gate.dtype in (torch.float32, torch.bfloat16, torch.float16)):
        if not _needs_grad(gate, up):
            return aten_fast.geglu_forward(gate, up, approximate)
        return _GeGLU.apply(gate, up, approximate)
    return F.gelu(gate, approximate=approximate) * up


def rms_norm(x, weight, eps, weight_offset=0.0):
    """rms_norm over the last dim with scale (weight + weight_offset), the
    scale formed in f32 (Gemma: weight_offset = 1)."""
    from .mojo_device.mojo_device_autograd import _FusedRMSNorm

    shape = (x.shape[-1],)
    if _on_mojo(x, weight) and aten_fast.rms_norm_inputs(x, shape, weight):
        if not _needs_grad(x, weight):
            return aten_fast.rms_norm_forward(x, shape, weight, float(eps), float(weight_offset))[0]
        return _FusedRMSNorm.apply(x, shape, weight, float(eps), float(weight_offset))
    return F.rms_norm(x, shape, weight.float() + weight_offset, eps)


def sliding_window_attention(q, k, v, window, *, sinks=0, scale=None):
    """Causal attention of q [B, H, T, D] over k, v [B, H_kv, T, D] with a
    sliding window and `sinks` first tokens that stay visible: query i sees key
    j <= i with i - j < window or j < sinks.  Query head h reads K/V head
    h // (H // H_kv); scale defaults to D ** -0.5.  Differentiable in q, k and
    v.  The scores of what is not visible are not computed, and no mask is
    held: F.scaled_dot_product_attention with a mask of
    masks.sliding_window_causal_mask runs the same kernels, but for bf16 and f16
    at head_dim 64 without sinks, where it keeps those of plain windows."""
    what = "sliding_window_attention"
    window, sinks = int(window), int(sinks)
    if window <= 0 or sinks < 0:
        raise ValueError(f"{what}: window {window} must be positive, sinks {sinks} not negative")
    if any(x.dim() != 4 for x in (q, k, v)) or k.shape != v.shape or q.shape[0] != k.shape[0] \
            or q.shape[2:] != k.shape[2:]:
        raise ValueError(f"{what}: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} must be"
                         " [batch, heads, tokens, head_dim] of the same batch, tokens and head_dim")
    if k.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f"{what}: {q.shape[1]} heads over {k.shape[1]} K/V heads")
    if not q.dtype == k.dtype == v.dtype or not q.device == k.device == v.device:
        raise TypeError(f"{what}: q, k and v must be of one dtype on one device")
    if scale is not None and not math.isfinite(float(scale)):
        raise ValueError(f"{what}: scale {scale} must be finite")
    t = q.shape[2]
    if _on_mojo(q, k, v) and q.numel():
        if q.dtype not in (torch.float32, torch.bfloat16, torch.float16) or q.shape[3] > 256:
            raise NotImplementedError(f"{what}: {q.dtype} with head_dim {q.shape[3]} is not supported"
                                      " (float32, bfloat16, float16, head_dim up to 256)")
        # (a window of all tokens too: plain causal attention would take its
        # row terms from the rounded output, dQ and dK of 6 tokens 3.3e-3 off
        # instead of 2.4e-3)
        window, sinks = min(window, t), min(sinks, t)
        if not _needs_grad(q, k, v):
            materialize_touched((q, k, v), None, False)
            return paged.on_device(q._device, aten_fast.attention_forward, q, k, v, True, window, scale, sinks)[0]
        from .mojo_device.mojo_device_autograd import _FusedAttention

        materialize_touched((q, k, v), None, False)
        return paged.on_device(q._device, _FusedAttention.apply, q, k, v, True, window, scale, sinks)
    if not q.numel():
        return q * 1.0
    return F.scaled_dot_product_attention(
        q, k, v, attn_mask=sliding_window_causal_mask(t, min(window, t), q.device, sinks=sinks), scale=scale, enable_gqa=True)


# ---------------------------------------------------------------------------
# paged key/value cache (torch_mojo_backend.kv_cache)
# ---------------------------------------------------------------------------
def _paged_check(what, cache, page_table, starts, counts, batch, **tensors):
    """The arguments that the cache's operations share."""
    for name, t, dims in (("page_table", page_table, 2), ("starts", starts, 1), ("counts", counts, 1)):
        if t is None and name == "counts":
            continue
        if t.dtype != torch.int32 or t.dim() != dims or t.shape[0] != batch:
            raise ValueError(f"{what}: {name} must be int32 with {dims} dimension{'s' * (dims > 1)} and {batch} rows,"
                             f" got {tuple(t.shape)} of {t.dtype}")
        if t.numel() and t.stride(-1) != 1 and t.shape[-1] > 1:
            raise ValueError(f"{what}: {name} must have unit stride")
    every = dict(tensors, page_table=page_table, starts=starts, counts=counts)
    for name, t in every.items():
        if t is None:
            continue
        if t.device != cache.device:
            raise ValueError(f"{what}: {name} is on {t.device}, the cache on {cache.device}")
        if cache.on_mojo != isinstance(t, TorchMojoTensor):
            raise ValueError(f"{what}: {name} and the cache must both be mojo tensors")
        if _needs_grad(t):
            raise NotImplementedError(f"{what} has no gradient: call it under torch.no_grad(), or detach {name}")


def _paged_rows(what, cache, name, t, heads, dtype):
    if t.dim() != 4 or t.shape[3] != cache.head_dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{what}: {name} must be [batch, {'heads' if heads is None else heads}, tokens,"
                         f" {cache.head_dim}], got {tuple(t.shape)}")
    if t.dtype not in (torch.float32, torch.bfloat16, torch.float16) or t.dtype != dtype:
        raise TypeError(f"{what}: {name} is of {t.dtype}, expected {dtype}")


def paged_append(cache, page_table, starts, k, v, cos=None, sin=None, *, q=None, counts=None):
    """Put the keys and values of new tokens into their pages: token t of
    sequence b (k, v [batch, kv_heads, tokens, head_dim]) goes to position
    starts[b] + t, page page_table[b, position // page_size]; tokens from
    counts[b] on are padding and are not written.  With cos and sin
    [positions, head_dim] (f32 or k's dtype) keys are turned by the angles of
    their positions, as `rotary_embedding` does, and so is q [batch, heads,
    tokens, head_dim], which is returned (zero at padding; None without q).

    One kernel.  A position outside the page table, a page that does not exist
    or a position outside cos raises IndexError (on the mojo device at the next
    device-to-host read) and is not written.  Two tokens of one call must not
    name the same slot; rows that are views of the pages are read before any
    is written."""
    if (paged.seqs_ok(cache, page_table, starts, counts) and paged.rows_ok(cache, k, page_table._shape[0])
            and paged.rows_ok(cache, v, page_table._shape[0], k) and k._shape[1] == cache.kv_heads and k._shape == v._shape
            and (cos is None) == (sin is None) == (q is None)
            and (cos is None or (type(cos) is type(sin) is TorchMojoTensor and cos._dtype is sin._dtype
                                 and (cos._dtype is torch.float32 or cos._dtype is k._dtype)
                                 and len(cos._shape) == 2 and cos._shape == sin._shape
                                 and cos._shape[1] == cache.head_dim and cache.head_dim % 16 == 0
                                 and cos._device == sin._device == k._device and paged.rows_ok(cache, q, k._shape[0], k)
                                 and q._shape[2] == k._shape[2] and q._shape[1]))
            and not _needs_grad(cos, sin)):
        return paged.append(cache, page_table, starts, k, v, cos, sin, q, counts)
    what = "paged_append"
    if k.dim() != 4:
        raise ValueError(f"{what}: k must be [batch, kv_heads, tokens, head_dim], got {tuple(k.shape)}")
    _paged_check(what, cache, page_table, starts, counts, k.shape[0], k=k, v=v, cos=cos, sin=sin, q=q)
    dtype = k.dtype if cache.bits == 4 else cache.dtype
    _paged_rows(what, cache, "k", k, cache.kv_heads, dtype)
    _paged_rows(what, cache, "v", v, cache.kv_heads, dtype)
    if v.shape != k.shape:
        raise ValueError(f"{what}: k is {tuple(k.shape)}, v {tuple(v.shape)}")
    if (cos is None) != (sin is None):
        raise ValueError(f"{what}: cos and sin come together")
    if cos is not None:
        if cos.dim() != 2 or cos.shape[1] != cache.head_dim or cos.shape != sin.shape:
            raise ValueError(f"{what}: cos and sin must be [positions, {cache.head_dim}], got {tuple(cos.shape)}"
                             f" and {tuple(sin.shape)}")
        if cos.dtype not in (torch.float32, k.dtype) or sin.dtype != cos.dtype:
            raise TypeError(f"{what}: cos and sin are of {cos.dtype} and {sin.dtype}, expected torch.float32 or {k.dtype}")
        if cache.head_dim % 16:
            raise ValueError(f"{what}: the rotation needs a head_dim that is a multiple of 16, not {cache.head_dim}")
    if q is not None:
        if cos is None:
            raise ValueError(f"{what}: q is taken with cos and sin")
        _paged_rows(what, cache, "q", q, None, dtype)
        if q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2] or q.shape[1] == 0:
            raise ValueError(f"{what}: q is {tuple(q.shape)}, k {tuple(k.shape)}")
    if cache.on_mojo:
        return paged.append(cache, page_table, starts, k, v, cos, sin, q, counts)
    return kv_cache.append_plain(cache, page_table, starts, k, v, cos, sin, q, counts)


def paged_gather(cache, page_table, starts, length, *, counts=None, dtype=None):
    """(k, v) [batch, kv_heads, length, head_dim]: the rows at positions
    starts[b] .. starts[b] + length - 1 back as values of dtype (the cache's,
    float32 of a 4-bit one), zero from counts[b] on."""
    what = "paged_gather"
    _paged_check(what, cache, page_table, starts, counts, page_table.shape[0] if page_table.dim() else 0)
    dtype = dtype or (torch.float32 if cache.bits == 4 else cache.dtype)
    if dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"{what}: values of {dtype} are not supported")
    length = int(length)
    if length < 0:
        raise ValueError(f"{what}: length {length}")
    if cache.on_mojo:
        return paged.gather(cache, page_table, starts, length, counts, dtype)
    return kv_cache.gather_plain(cache, page_table, starts, length, counts, dtype)


def paged_attention(q, cache, page_table, starts, *, counts=None, window=0, sinks=0, scale=None):
    """Attention of new tokens over their sequences' pages, which hold the
    tokens' own keys and values already: the query t of sequence b (q [batch,
    heads, tokens, head_dim]) at position p = starts[b] + t sees key j <= p and,
    with a window > 0, only p - j < window or j < sinks.  Query head h reads
    K/V head h // (heads // kv_heads).  Queries from counts[b] on are padding:
    their rows are zero, as is a row that sees no key.  scale defaults to
    head_dim ** -0.5.

    A page that does not exist raises IndexError (on the mojo device at the
    next device-to-host read) and counts as hidden.  Pages that no query sees
    are not looked up: the table may say anything of pages that lie behind a
    sequence's last token, or between its sinks and its window.  What lies in
    rows that no query sees is never used; a NaN or an infinity in the value of
    a row that some query of the sequence sees may reach the call's others, as
    0 * NaN does in the plain formula."""
    if (paged.seqs_ok(cache, page_table, starts, counts) and paged.rows_ok(cache, q, page_table._shape[0])
            and q._shape[1] and q._shape[1] % cache.kv_heads == 0 and type(window) is type(sinks) is int
            and 0 <= window < 2 ** 31 and 0 <= sinks < 2 ** 31 and scale is None):
        return paged.attention(q, cache, page_table, starts, counts, window, sinks, cache.scale)
    what = "paged_attention"
    if q.dim() != 4:
        raise ValueError(f"{what}: q must be [batch, heads, tokens, head_dim], got {tuple(q.shape)}")
    _paged_check(what, cache, page_table, starts, counts, q.shape[0], q=q)
    _paged_rows(what, cache, "q", q, None, q.dtype if cache.bits == 4 else cache.dtype)
    if q.shape[1] == 0 or q.shape[1] % cache.kv_heads:
        raise ValueError(f"{what}: {q.shape[1]} heads over {cache.kv_heads} K/V heads")
    window, sinks = int(window), int(sinks)
    if window < 0 or sinks < 0:
        raise ValueError(f"{what}: window {window} and sinks {sinks} must not be negative")
    window, sinks = min(window, 2 ** 31 - 1), min(sinks, 2 ** 31 - 1)  # past every position
    scale = cache.scale if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"{what}: scale {scale} must be finite")
    if cache.on_mojo:
        return paged.attention(q, cache, page_table, starts, counts, window, sinks, scale)
    return kv_cache.attention_plain(q, cache, page_table, starts, counts, window, sinks, scale)
