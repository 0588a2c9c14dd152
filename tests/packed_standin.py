"""The entry points of packed sequences, rotary positions and token
log-probabilities for the host stand-in of the library, over host memory with the
plain formulas of torch_mojo_backend.packing, rotary and logprobs.  A plan here
is the offsets, behind whether they are sound."""

from __future__ import annotations

import ctypes
import itertools
import types

import torch

from host_standin import DT, HostStandIn, _val, dense, view
from torch_mojo_backend import logprobs, packing, rotary


def _flag(error):
    if error:
        ctypes.c_int32.from_address(_val(error)).value = 1


def _plan(self, plan, size, positions, offsets, n, tokens, error, stream):
    assert size >= 16 * (n + 2)
    at = dense(_val(offsets), torch.int32, (n + 1,)).tolist()
    good = at[0] >= 0 and at[-1] <= tokens and all(b >= a for a, b in itertools.pairwise(at))
    if not good:
        _flag(error)
        at = [0] * (n + 1)
    dense(_val(plan), torch.int32, (n + 1,)).copy_(torch.tensor(at, dtype=torch.int32))
    where = dense(_val(positions), torch.int32, (tokens,))
    where.zero_()
    for a, b in itertools.pairwise(at):
        where[a:b] = torch.arange(b - a, dtype=torch.int32)
    return 0


def _seqs(plan, n):
    return types.SimpleNamespace(_offsets=dense(_val(plan), torch.int32, (n + 1,)).tolist())


def _rows(ptr, dt, t, h, d, th):
    return view(_val(ptr), DT[dt], (t, h, d), (*th, 1))


def _fwd(self, o, o_th, o_low, lse, q, q_th, k, k_th, v, v_th, plan, n, t, h, hk, d, scale, window, dt, stream):
    qq, kk, vv = (_rows(p, dt, t, m, d, s).double() for p, s, m in ((q, q_th, h), (k, k_th, hk), (v, v_th, hk)))
    out = packing.attention_plain(qq, kk, vv, _seqs(plan, n), window, scale)
    oo = _rows(o, dt, t, h, d, o_th)
    oo.copy_(out)
    if _val(o_low):
        _rows(o_low, dt, t, h, d, o_th).copy_(out - oo.double())
    dense(_val(lse), torch.float32, (h, t)).zero_()
    return 0


def _bwd(self, dq, dq_th, dk, dk_th, dv, dv_th, do, do_th, q, q_th, k, k_th, v, v_th, o, o_th, o_low, lse, plan, n, t, h, hk,
         d, scale, window, dt, ws, nws, stream):
    assert ws and nws >= 64
    qq, kk, vv, gg = (_rows(p, dt, t, m, d, st).double() for p, st, m in ((q, q_th, h), (k, k_th, hk), (v, v_th, hk), (do, do_th, h)))
    grads = [torch.zeros_like(x) for x in (qq, kk, vv)]
    group = h // hk
    for a, b in itertools.pairwise(_seqs(plan, n)._offsets):
        i = torch.arange(b - a)
        hidden = (i[None] > i[:, None]) | ((i[:, None] - i[None] >= window) if window else False)
        x, dy = (y[a:b].transpose(0, 1) for y in (qq, gg))
        ks, vs = (y[a:b].transpose(0, 1).repeat_interleave(group, 0) for y in (kk, vv))
        p = torch.softmax((x @ ks.mT * scale).masked_fill(hidden, float("-inf")), -1)
        ds = p * (dy @ vs.mT - (dy * (p @ vs)).sum(-1, keepdim=True)) * scale
        grads[0][a:b] = (ds @ ks).transpose(0, 1)
        for y, z in ((grads[1], ds.mT @ x), (grads[2], p.mT @ dy)):
            y[a:b] = z.reshape(hk, group, b - a, d).sum(1).transpose(0, 1)
    for p, st, m, g in ((dq, dq_th, h, grads[0]), (dk, dk_th, hk, grads[1]), (dv, dv_th, hk, grads[2])):
        _rows(p, dt, t, m, d, st).copy_(g)
    return 0


def _rope(self, qo, qo_bht, q, q_bht, h, ko, ko_bht, k, k_bht, hk, positions, pdt, pst, freq, b, t, d, turned, laced, scale,
          inverse, dt, stream):
    pos = view(_val(positions), DT[pdt], (b, t), (pst, 1))
    f = dense(_val(freq), torch.float64, (turned // 2,))
    for out, out_st, x, st, m in ((qo, qo_bht, q, q_bht, h), (ko, ko_bht, k, k_bht, hk)):
        if m:
            y = rotary.turn_plain(view(_val(x), DT[dt], (b, m, t, d), (*st, 1)), pos, f, bool(laced), scale, bool(inverse))
            view(_val(out), DT[dt], (b, m, t, d), (*out_st, 1)).copy_(y)
    return 0


def _lp_fwd(self, picked, spread, stats, best, order, x, dt, ld, tokens, n, c, top, ignore, error, ws, nws, stream):
    xx = view(_val(x), DT[dt], (n, c), (ld, 1))
    tk = dense(_val(tokens), torch.int64, (n,)).clone() if tokens else None
    if tk is not None:
        bad = (tk != ignore) & ((tk < 0) | (tk >= c))
        if bad.any():
            _flag(error)
            tk[bad] = ignore
    got = logprobs.plain(xx, tk, top, bool(spread), ignore)
    for p, shape, value in ((picked, (n,), got.logprobs), (spread, (n,), got.entropy), (best, (n, top), got.top_logprobs)):
        if p:
            dense(_val(p), torch.float32, shape).copy_(value)
    if order:
        dense(_val(order), torch.int64, (n, top)).copy_(got.top_tokens)
    return 0


def _lp_bwd(self, dx, ld_dx, x, dt, ld, stats, spread, tokens, order, top, d_picked, d_spread, d_best, n, c, ignore, stream):
    logp = torch.log_softmax(view(_val(x), DT[dt], (n, c), (ld, 1)).double(), -1)
    p, ones = logp.exp(), torch.zeros(n, c, dtype=torch.float64)
    if d_picked:
        tk = dense(_val(tokens), torch.int64, (n,))
        good = (tk != ignore) & (tk >= 0) & (tk < c)
        ones.scatter_add_(1, (tk * good)[:, None], (dense(_val(d_picked), torch.float32, (n,)).double() * good)[:, None])
    if d_best:
        ones.scatter_add_(1, dense(_val(order), torch.int64, (n, top)), dense(_val(d_best), torch.float32, (n, top)).double())
    g = ones - p * ones.sum(-1, keepdim=True)
    if d_spread:
        h = dense(_val(spread), torch.float32, (n,)).double()[:, None]
        g = g - p * (logp.clamp(min=-1e4) + h) * dense(_val(d_spread), torch.float32, (n,)).double()[:, None]
    out = view(_val(dx), DT[dt], (n, ld_dx), (ld_dx, 1))
    out.zero_()
    out[:, :c] = g
    return 0


HostStandIn.mi355x_packed_plan_bytes = lambda self, n, t: 16 * (n + 2)
HostStandIn.mi355x_packed_plan = _plan
HostStandIn.mi355x_packed_attn_fwd = _fwd
HostStandIn.mi355x_packed_attn_bwd_workspace_bytes = lambda self, *a: 64
HostStandIn.mi355x_packed_attn_bwd = _bwd
HostStandIn.mi355x_rope_at = _rope
HostStandIn.mi355x_token_logprobs_workspace_bytes = lambda self, *a: 0
HostStandIn.mi355x_token_logprobs_fwd = _lp_fwd
HostStandIn.mi355x_token_logprobs_bwd = _lp_bwd
