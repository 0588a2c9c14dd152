"""Sliding-window attention with sinks on the MI355X against f64, forward and
backward, over types, head layouts, lengths and masks."""

import pytest
import torch
import torch.nn.functional as F

import window_cases
from paged_cases import check
from torch_mojo_backend import ops
from torch_mojo_backend.masks import sliding_window_causal_mask

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _mojo(mojo):
    return mojo


def run(x, window, sinks, scale=None, mask=None):
    q, k, v = (y.transpose(1, 2).contiguous().to("mojo").transpose(1, 2).requires_grad_() for y in x[:3])
    if mask is not None:
        out = F.scaled_dot_product_attention(q, k, v, attn_mask=mask, scale=scale, enable_gqa=True)
    else:
        out = ops.sliding_window_attention(q, k, v, window, sinks=sinks, scale=scale)
    out.backward(x[3].to("mojo"))
    return {"out": out, "dq": q.grad, "dk": k.grad, "dv": v.grad}


def compare(got, want):
    for name, value in got.items():
        check(value, *want[name], name)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("d,h,hk", [(64, 2, 2), (128, 4, 1), (256, 4, 2), (96, 2, 2), (20, 3, 1)])
@pytest.mark.parametrize("t,window,sinks", [(1, 8, 1), (63, 1, 1), (65, 16, 3), (200, 64, 4), (333, 40, 70),
                                            (500, 100, 1), (257, 300, 4), (130, 64, 129)])
def test_forward_and_backward(dtype, d, h, hk, t, window, sinks):
    x = window_cases.inputs(2, h, hk, t, d, dtype)
    compare(run(x, window, sinks), window_cases.expected(*x, window, sinks))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_by_mask_is_the_same(dtype):
    x = window_cases.inputs(1, 4, 2, 300, 64, dtype)
    a, b = run(x, 32, 5), run(x, 32, 5, mask=sliding_window_causal_mask(300, 32, "mojo", sinks=5))
    for n in a:
        assert torch.equal(a[n].detach().cpu(), b[n].detach().cpu()), n


@pytest.mark.parametrize("dtype,d,hk", [(BF, 64, 4), (BF, 256, 1), (F32, 64, 4)])
def test_without_sinks(dtype, d, hk):
    x = window_cases.inputs(1, 4, hk, 400, d, dtype)
    compare(run(x, 48, 0), window_cases.expected(*x, 48, 0))


@pytest.mark.parametrize("scale", [-0.2, 1.0])
def test_scales(scale):
    x = window_cases.inputs(1, 2, 1, 190, 128, BF)
    compare(run(x, 50, 4, scale), window_cases.expected(*x, 50, 4, scale))


@pytest.mark.parametrize("d,h,hk", [(64, 2, 2), (256, 2, 1)])
def test_long_sequences(d, h, hk):
    x = window_cases.inputs(1, h, hk, 2500, d, BF)
    compare(run(x, 300, 4), window_cases.expected(*x, 300, 4))


def test_results_repeat():
    x = window_cases.inputs(2, 4, 2, 700, 64, BF)
    a, b = run(x, 100, 4), run(x, 100, 4)
    for n in a:
        assert torch.equal(a[n].detach().cpu(), b[n].detach().cpu()), n


def test_broadcast_gradient_and_shared_leaf():
    """One tensor as q, k and v, and a gradient that is an expanded scalar."""
    x = window_cases.inputs(1, 2, 2, 100, 64, F32)[0]
    leaf = x.to("mojo").requires_grad_()
    ops.sliding_window_attention(leaf, leaf, leaf, 20, sinks=2).sum().backward()
    want = window_cases.expected(x, x, x, torch.ones_like(x), 20, 2)
    check(leaf.grad, sum(want[n][0] for n in ("dq", "dk", "dv")),
          sum(want[n][1] for n in ("dq", "dk", "dv")) + 2.0 ** -22 * 4)


@pytest.mark.parametrize("d,h,hk", [(32, 2, 2), (32, 3, 1), (128, 4, 2), (256, 6, 3)])
@pytest.mark.parametrize("t,window,sinks", [(64, 1, 1), (129, 31, 17), (300, 64, 40), (777, 100, 4)])
def test_f32_heads(d, h, hk, t, window, sinks):
    x = window_cases.inputs(1, h, hk, t, d, F32)
    compare(run(x, window, sinks), window_cases.expected(*x, window, sinks))


@pytest.mark.parametrize("dtype,d,hk", [(BF, 64, 2), (BF, 128, 1), (HF, 256, 2), (F32, 64, 1), (F32, 256, 2), (F32, 80, 1)])
def test_many_sinks(dtype, d, hk):
    """More sinks than one block of keys has, a last block with a few of them, and all of them."""
    for t, window, sinks in ((600, 70, 300), (450, 33, 129), (300, 20, 2 ** 40)):
        x = window_cases.inputs(1, 2, hk, t, d, dtype)
        compare(run(x, window, sinks), window_cases.expected(*x, window, min(sinks, t)))


@pytest.mark.parametrize("dtype,d", [(BF, 64), (HF, 128), (F32, 64), (BF, 256)])
def test_strides_and_alignment(dtype, d):
    """Rows of one packed projection, at odd offsets, heads first, and an expanded gradient."""
    h, t = 2, 150
    x = window_cases.inputs(2, h, h, t, d, dtype)
    want = window_cases.expected(*x, 40, 3)
    packed = torch.cat([y.transpose(1, 2).reshape(2, t, h * d) for y in x[:3]], dim=-1).to("mojo").requires_grad_()
    q, k, v = (y.view(2, t, h, d).transpose(1, 2) for y in packed.split(h * d, dim=-1))
    out = ops.sliding_window_attention(q, k, v, 40, sinks=3)
    out.backward(x[3].to("mojo"))
    got = [y.view(2, t, h, d).transpose(1, 2) for y in packed.grad.cpu().split(h * d, dim=-1)]
    compare(dict(zip(("out", "dq", "dk", "dv"), (out, *got))), want)

    def odd(y):  # one element past an aligned address, rows of d + 1
        wide = torch.zeros(2, h, t, d + 1, dtype=dtype)
        wide[..., 1:] = y
        return wide.to("mojo")[..., 1:]

    leaves = [odd(y).detach().requires_grad_() for y in x[:3]]
    out = ops.sliding_window_attention(*leaves, 40, sinks=3)
    out.backward(odd(x[3]))
    compare(dict(zip(("out", "dq", "dk", "dv"), (out, *(y.grad for y in leaves)))), want)

    ones = torch.ones(1, dtype=dtype)
    leaves = [y.contiguous().to("mojo").requires_grad_() for y in x[:3]]
    out = ops.sliding_window_attention(*leaves, 40, sinks=3)
    out.backward(ones.to("mojo").expand(2, h, t, d))
    want = window_cases.expected(*x[:3], torch.ones(2, h, t, d, dtype=dtype), 40, 3)
    compare(dict(zip(("out", "dq", "dk", "dv"), (out, *(y.grad for y in leaves)))), want)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_hidden_numbers_stay_hidden(dtype):
    """NaN in a row of keys and values reaches no query whose tiles lie elsewhere."""
    x = window_cases.inputs(1, 2, 2, 400, 64, dtype)
    want = window_cases.expected(*x, 30, 2)["out"]
    k, v = x[1].clone(), x[2].clone()
    k[:, :, 200] = float("nan")
    v[:, :, 200] = float("nan")
    out = ops.sliding_window_attention(x[0].to("mojo"), k.to("mojo"), v.to("mojo"), 30, sinks=2)
    keep = torch.ones(400, dtype=torch.bool)
    keep[128:320] = False  # rows that share a 64-key tile with key 200: 192 .. 255 + 30, in blocks of 128 queries
    check(out.cpu()[:, :, keep], want[0][:, :, keep.numpy()], want[1][:, :, keep.numpy()])


@pytest.mark.parametrize("dtype,d", [(BF, 64), (BF, 256), (HF, 128), (F32, 64), (F32, 96)])
def test_captured_and_replayed(kernels, dtype, d):
    """Forward and backward through the C entry points, in a graph whose inputs
    change between the replays."""
    import ctypes

    from torch_mojo_backend.eager_kernels import check as ok

    b, h, hk, t, window, sinks = 1, 4, 2, 700, 100, 4
    code = {F32: 0, BF: 1, HF: 2}[dtype]
    make = lambda n: torch.empty(b, t, n, d, dtype=dtype, device="cuda").transpose(1, 2)  # noqa: E731
    q, k, v, do, o, dq, dk, dv = make(h), make(hk), make(hk), make(h), make(h), make(h), make(hk), make(hk)
    low = torch.full_like(o, float("nan"))
    lse = torch.empty(b, h, t, device="cuda")
    ws = kernels.mi355x_attn_bwd_sink_workspace_bytes(b, h, hk, t, t, d, window, sinks)
    hold = torch.empty(ws, dtype=torch.uint8, device="cuda")
    st = lambda x: (ctypes.c_int64 * 3)(*x.stride()[:3])  # noqa: E731
    at = lambda *xs: [y for x in xs for y in (x.data_ptr(), st(x))]  # noqa: E731

    def step(stream):
        ok("forward", kernels.mi355x_attn_fwd_sink(o.data_ptr(), st(o), low.data_ptr(), lse.data_ptr(), *at(q, k, v), b, h, hk, t, t, d,
                                                   d ** -0.5, window, sinks, code, stream))
        ok("backward", kernels.mi355x_attn_bwd_sink(*at(dq, dk, dv, do, q, k, v, o), low.data_ptr(), lse.data_ptr(), b, h, hk, t, t, d,
                                                    d ** -0.5, window, sinks, code, hold.data_ptr(), ws, stream))

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    for x in (q, k, v, do):
        x.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step(side.cuda_stream)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            step(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for seed in range(3):
        x = window_cases.inputs(b, h, hk, t, d, dtype, seed=seed)
        for dst, src in zip((q, k, v, do), x):
            dst.copy_(src.cuda())
        hold.fill_(255)  # what is left there is not used
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        compare({"out": o, "dq": dq, "dk": dk, "dv": dv}, window_cases.expected(*x, window, sinks))


@pytest.mark.parametrize("dtype,d", [(BF, 64), (HF, 128), (BF, 256), (F32, 64), (F32, 256), (F32, 40)])
@pytest.mark.parametrize("sq,skv,window,sinks", [(300, 100, 50, 3), (300, 100, 50, 0), (90, 400, 30, 2), (1, 70, 5, 1)])
def test_more_queries_or_more_keys(kernels, dtype, d, sq, skv, window, sinks):
    """The C entry points take lengths that differ: queries that see nothing give
    zeros, and so do the gradients of keys that nothing sees."""
    import ctypes

    import numpy as np

    from paged_cases import np64
    from torch_mojo_backend.eager_kernels import check as ok

    n = max(sq, skv)
    x = window_cases.inputs(1, 2, 1, n, d, dtype)
    q, do = (y[:, :, :sq] for y in (x[0], x[3]))
    k, v = (y[:, :, :skv] for y in x[1:3])
    dev = [y.contiguous().cuda() for y in (q, k, v, do)]
    o, dq, dk, dv = (torch.full_like(dev[i], float("nan")) for i in (0, 0, 1, 2))
    lse = torch.empty(1, 2, sq, device="cuda")
    st = lambda y: (ctypes.c_int64 * 3)(*y.stride()[:3])  # noqa: E731
    at = lambda *ys: [z for y in ys for z in (y.data_ptr(), st(y))]  # noqa: E731
    code = {F32: 0, BF: 1, HF: 2}[dtype]
    ws = kernels.mi355x_attn_bwd_sink_workspace_bytes(1, 2, 1, sq, skv, d, window, sinks)
    hold = torch.full((ws,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ok("forward", kernels.mi355x_attn_fwd_sink(o.data_ptr(), st(o), None, lse.data_ptr(), *at(*dev[:3]), 1, 2, 1, sq, skv, d,
                                               d ** -0.5, window, sinks, code, None))
    ok("backward", kernels.mi355x_attn_bwd_sink(*at(dq, dk, dv, dev[3], *dev[:3], o), None, lse.data_ptr(), 1, 2, 1, sq, skv, d,
                                                d ** -0.5, window, sinks, code, hold.data_ptr(), ws, None))
    torch.cuda.synchronize()
    # the same with n queries and n keys, those that are not there without weight or gradient
    qn, kn, vn, dn = (np64(y) for y in x)
    dn[:, :, sq:] = 0
    i, j = np.arange(n)[:, None], np.arange(n)[None]
    seen = (j <= i) & ((i - j < window) | (j < sinks)) & (j < skv)
    s = np.where(seen, d ** -0.5 * (qn @ kn.swapaxes(-1, -2)), -np.inf)
    top = np.where(seen.any(-1), s.max(-1), 0.0)[..., None]
    p = np.where(seen, np.exp(s - top), 0.0)
    p = p / np.maximum(p.sum(-1, keepdims=True), 1e-300)
    on = p @ vn
    ds = p * (dn @ vn.swapaxes(-1, -2) - (dn * on).sum(-1, keepdims=True))
    want = {"out": on[:, :, :sq], "dq": (d ** -0.5 * ds @ kn)[:, :, :sq],
            "dk": (d ** -0.5 * ds.swapaxes(-1, -2) @ qn).sum(1, keepdims=True)[:, :, :skv],
            "dv": (p.swapaxes(-1, -2) @ dn).sum(1, keepdims=True)[:, :, :skv]}
    bound = window_cases.expected(*x, window, max(sinks, 1))
    for name, got in (("out", o), ("dq", dq), ("dk", dk), ("dv", dv)):
        assert torch.isfinite(got).all(), name
        # at most the largest bound of the square case, whose sums have no fewer terms
        check(got, want[name], np.full(want[name].shape, bound[name][1].max()), name)
    empty = ~seen.any(-1)[:sq]
    assert (np64(o)[:, :, empty] == 0).all() and (np64(dq)[:, :, empty] == 0).all()


@pytest.mark.parametrize("dtype,d", [(BF, 64), (HF, 128), (BF, 256), (BF, 96)])
def test_what_rounding_takes_from_the_output_is_kept(dtype, d):
    """Two visible keys a query: dP - D is a small difference, and D from the
    rounded output alone makes dQ and dK worse."""
    from paged_cases import np64
    from torch_mojo_backend.eager_kernels import aten_fast

    x = window_cases.inputs(1, 2, 2, 300, d, dtype)
    want = window_cases.expected(*x, 1, 1)
    q, k, v, do = (y.to("mojo") for y in x)
    errors = []
    for low in (None, aten_fast.alloc_bthd(1, 2, 300, d, dtype, q._device)):
        out, lse = aten_fast.attention_forward(q, k, v, True, 1, None, 1, low)
        dq, dk, _ = aten_fast.attention_backward(do, q, k, v, out, lse, True, 1, None, 1, low)
        errors.append([abs(np64(g) - want[n][0]).sum() for g, n in ((dq, "dq"), (dk, "dk"))])
        if low is not None:  # of half a step of the output at most
            assert (abs(np64(low)) <= window_cases.STEP[dtype] * abs(np64(out)) + 2.0 ** -25).all()
            both = np64(out) + np64(low)
            assert abs(both - want["out"][0]).sum() < abs(np64(out) - want["out"][0]).sum()
    assert all(kept < 0.85 * alone for alone, kept in zip(*errors)), errors


@pytest.mark.parametrize("dtype,d,hk", [(BF, 64, 2), (HF, 128, 1), (BF, 256, 1), (F32, 64, 2), (F32, 128, 1)])
@pytest.mark.parametrize("t,window,sinks", [(2300, 40, 150), (1700, 100, 190), (1500, 64, 20), (1500, 1, 250), (700, 300, 400),
                                            (701, 300, 400)])
def test_partials_of_many_sinks(dtype, d, hk, t, window, sinks):
    """Last blocks of sinks of one wave, of two, of more, with several chunks of
    queries; sinks and window that hide nothing, and one key."""
    x = window_cases.inputs(1, 2, hk, t, d, dtype)
    compare(run(x, window, sinks), window_cases.expected(*x, window, sinks))


@pytest.mark.parametrize("dtype,d,hk", [(BF, 64, 2), (F32, 256, 1)])
def test_a_gradient_of_the_gradient_is_refused(dtype, d, hk):
    x = window_cases.inputs(1, 2, hk, 90, d, dtype)
    q, k, v = (y.to("mojo").requires_grad_() for y in x[:3])
    out = ops.sliding_window_attention(q, k, v, 20, sinks=2)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), x[3].to("mojo"), create_graph=True)
    compare({"out": out, "dq": dq, "dk": dk, "dv": dv}, window_cases.expected(*x, 20, 2))
    with pytest.raises(RuntimeError, match="second time"):
        (out.float().sum() + (dk.float() * dk.float()).sum()).backward()


@pytest.mark.parametrize("dtype,d,h,hk", [(F32, 64, 2, 2), (F32, 32, 4, 2), (F32, 256, 2, 1), (BF, 128, 4, 1), (HF, 256, 2, 2), (BF, 96, 2, 1),
                                          (BF, 64, 2, 2), (HF, 64, 4, 2)])
@pytest.mark.parametrize("t,window", [(300, 32), (130, 129), (130, 200)])
def test_masks_without_sinks(dtype, d, h, hk, t, window):
    """The kernels of ops.sliding_window_attention, but for 16-bit types at head_dim 64."""
    x = window_cases.inputs(1, h, hk, t, d, dtype)
    got = run(x, window, 0, mask=sliding_window_causal_mask(t, window, "mojo"))
    compare(got, window_cases.expected(*x, window, 0))
    if t > window and (dtype is F32 or d != 64):
        op = run(x, window, 0)
        for n in op:
            assert torch.equal(op[n].detach().cpu(), got[n].detach().cpu()), n


@pytest.mark.parametrize("dtype,d,h,hk", [(BF, 64, 8, 8), (HF, 128, 8, 2), (BF, 256, 4, 4), (BF, 96, 8, 4)])
@pytest.mark.parametrize("t,window", [(3, 3), (3, 100), (2, 2 ** 40)])
def test_windows_of_all_tokens_keep_what_rounding_takes(dtype, d, h, hk, t, window):
    """As narrow ones do: with few keys a row the row terms dO . O decide."""
    from paged_cases import np64
    from torch_mojo_backend.eager_kernels import aten_fast

    x = window_cases.inputs(8, h, hk, t, d, dtype)
    want = window_cases.expected(*x, t, 0)
    got = run(x, window, 4)
    compare(got, want)
    q, k, v, do = (y.to("mojo") for y in x)
    out, lse = aten_fast.attention_forward(q, k, v, True, t, None, 0, None)
    alone = aten_fast.attention_backward(do, q, k, v, out, lse, True, t, None, 0, None)
    for n, a in zip(("dq", "dk"), alone):
        assert abs(np64(got[n]) - want[n][0]).sum() < 0.85 * abs(np64(a) - want[n][0]).sum(), n
