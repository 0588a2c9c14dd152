"""The paged cache's entry points for the host stand-in of the library, over
host memory with the plain formulas of torch_mojo_backend.kv_cache."""

from __future__ import annotations

import ctypes
import types

import torch

from host_standin import DT, HostStandIn, _val, view
from torch_mojo_backend import kv_cache


def _cache(c):
    n, hk, page, d = c.num_pages, c.kv_heads, c.page_size, c.d
    out = types.SimpleNamespace(num_pages=n, kv_heads=hk, page_size=page, head_dim=d, bits=c.bits)
    four = c.bits == 4
    for name in "kv":
        strides = tuple(getattr(c, name + "_phs"))
        dt, width = (torch.uint8, d // 2) if four else (DT[c.dtype], d)
        setattr(out, name, view(getattr(c, name), dt, (n, hk, page, width), (*strides, 1)))
        s = tuple(getattr(c, name + "s_phs"))
        setattr(out, name + "_scales", view(getattr(c, name + "_scales"), torch.float16, (n, hk, page, d // 32, 2),
                                            (*s, 2, 1)) if four else None)
    return out


def _ints(ptr, shape, strides):
    return view(_val(ptr), torch.int32, shape, strides)


def _run(error, call):
    try:
        return call()
    except IndexError:
        ctypes.c_int32.from_address(_val(error)).value = 1
        return None


def _rows(ptr, dt, shape, bht):
    return view(_val(ptr), dt, shape, (*bht, 1))


def _append(self, c, table, tst, width, starts, counts, k, k_bht, v, v_bht, qo, qo_bht, q, q_bht, cos, sin, rdt, rlen,
            b, h, t, dt, error, stream):
    if b * t == 0:
        return 0
    tab, st = _ints(table, (b, width), (tst, 1)), _ints(starts, (b,), (1,))
    cn = _ints(counts, (b,), (1,)) if counts else None
    kk, vv = (_rows(p, DT[dt], (b, c.kv_heads, t, c.d), s) for p, s in ((k, k_bht), (v, v_bht)))
    qq = _rows(q, DT[dt], (b, h, t, c.d), q_bht) if q else None
    cs = [view(_val(x), DT[rdt], (rlen, c.d), (c.d, 1)) for x in (cos, sin)] if cos else [None, None]
    out = _run(error, lambda: kv_cache.append_plain(_cache(c), tab, st, kk, vv, *cs, qq, cn))
    if q and out is not None:
        _rows(qo, DT[dt], (b, h, t, c.d), qo_bht).copy_(out)
    return 0


def _gather(self, k, k_bht, v, v_bht, c, table, tst, width, starts, counts, b, t, dt, error, stream):
    if b * t == 0:
        return 0
    tab, st = _ints(table, (b, width), (tst, 1)), _ints(starts, (b,), (1,))
    cn = _ints(counts, (b,), (1,)) if counts else None
    got = _run(error, lambda: kv_cache.gather_plain(_cache(c), tab, st, t, cn, DT[dt]))
    for p, s, x in zip((k, v), (k_bht, v_bht), got or ()):
        _rows(p, DT[dt], (b, c.kv_heads, t, c.d), s).copy_(x)
    return 0


def _attn(self, o, o_bht, q, q_bht, c, table, tst, width, starts, counts, b, h, t, scale, window, sinks, dt, ws, nws,
          error, stream):
    if b * t == 0:
        return 0
    assert ws and nws >= 64
    tab, st = _ints(table, (b, width), (tst, 1)), _ints(starts, (b,), (1,))
    cn = _ints(counts, (b,), (1,)) if counts else None
    qq = _rows(q, DT[dt], (b, h, t, c.d), q_bht)
    got = _run(error, lambda: kv_cache.attention_plain(qq, _cache(c), tab, st, cn, window, sinks, scale))
    if got is not None:
        _rows(o, DT[dt], (b, h, t, c.d), o_bht).copy_(got)
    return 0


HostStandIn.mi355x_paged_append = _append
HostStandIn.mi355x_paged_gather = _gather
HostStandIn.mi355x_paged_attn = _attn
HostStandIn.mi355x_paged_attn_workspace_bytes = lambda self, *a: 64


def _attn_fwd_sink(self, o, o_bhs, o_low, lse, q, q_bhs, k, k_bhs, v, v_bhs, b, h, hk, sq, skv, d, scale, window, sinks, dt,
                   stream):
    qq = _rows(q, DT[dt], (b, h, sq, d), q_bhs).float()
    kk, vv = (_rows(p, DT[dt], (b, hk, skv, d), s).float().repeat_interleave(h // hk, 1)
              for p, s in ((k, k_bhs), (v, v_bhs)))
    i, j = torch.arange(sq)[:, None], torch.arange(skv)[None, :]
    s = (qq @ kk.mT * scale).masked_fill((j > i) | ((i - j >= window) & (j >= sinks)), float("-inf"))
    view(_val(lse), torch.float32, (b, h, sq), (h * sq, sq, 1)).copy_(torch.logsumexp(s, -1))
    x, oo = torch.softmax(s, -1) @ vv, _rows(o, DT[dt], (b, h, sq, d), o_bhs)
    oo.copy_(x)
    if _val(o_low):
        _rows(o_low, DT[dt], (b, h, sq, d), o_bhs).copy_(x - oo.float())
    return 0


def _attn_bwd_sink(self, dq, dq_bhs, dk, dk_bhs, dv, dv_bhs, do, do_bhs, q, q_bhs, k, k_bhs, v, v_bhs, o, o_bhs, o_low,
                   lse, b, h, hk, sq, skv, d, scale, window, sinks, dt, ws, nws, stream):
    assert ws and nws >= 64
    low = _rows(o_low, DT[dt], (b, h, sq, d), o_bhs).float() if _val(o_low) else 0.0
    qq, gg, oo = (_rows(p, DT[dt], (b, h, sq, d), s).float() for p, s in ((q, q_bhs), (do, do_bhs), (o, o_bhs)))
    kk, vv = (_rows(p, DT[dt], (b, hk, skv, d), s).float().repeat_interleave(h // hk, 1)
              for p, s in ((k, k_bhs), (v, v_bhs)))
    i, j = torch.arange(sq)[:, None], torch.arange(skv)[None, :]
    s = (qq @ kk.mT * scale).masked_fill((j > i) | ((i - j >= window) & (j >= sinks)), float("-inf"))
    p = torch.exp(s - view(_val(lse), torch.float32, (b, h, sq, 1), (h * sq, sq, 1, 1)))
    ds = p * (gg @ vv.mT - (gg * (oo + low)).sum(-1, keepdim=True)) * scale
    grads = (ds @ kk, *(x.reshape(b, hk, h // hk, skv, d).sum(2) for x in (ds.mT @ qq, p.mT @ gg)))
    for p, s, x in zip((dq, dk, dv), (dq_bhs, dk_bhs, dv_bhs), grads):
        _rows(p, DT[dt], tuple(x.shape), s).copy_(x)
    return 0


HostStandIn.mi355x_attn_fwd_sink = _attn_fwd_sink
HostStandIn.mi355x_attn_bwd_sink = _attn_bwd_sink
HostStandIn.mi355x_attn_bwd_sink_workspace_bytes = lambda self, *a: 64
