"""Sliding-window attention with sinks off the GPU: against f64, through the
mask and through the function, its gradients and refusals."""

import pytest
import torch
import torch.nn.functional as F

import paged_standin  # noqa: F401
import window_cases
from paged_cases import check
from torch_mojo_backend import ops
from torch_mojo_backend.masks import sliding_window_causal_mask, window_and_sinks_of, window_of


@pytest.fixture(params=["cpu", "mojo"])
def device(request, mojo):
    if request.param == "mojo" and mojo != "host":
        pytest.skip("the stand-in is for machines without a GPU")
    return request.param


def leaf(x, device):
    return x.detach().to(device).requires_grad_()


@pytest.mark.parametrize("t,window,sinks", [(1, 4, 2), (9, 3, 2), (9, 3, 0), (9, 9, 2), (9, 100, 5), (9, 1, 1), (9, 2, 30)])
@pytest.mark.parametrize("by_mask", [False, True])
def test_forward_and_backward(device, t, window, sinks, by_mask):
    x = window_cases.inputs(2, 4, 2, t, 16, torch.float32)
    q, k, v = (leaf(y, device) for y in x[:3])
    if by_mask:
        mask = sliding_window_causal_mask(t, window, device, sinks=sinks)
        out = F.scaled_dot_product_attention(q, k, v, attn_mask=mask, enable_gqa=True)
    else:
        out = ops.sliding_window_attention(q, k, v, window, sinks=sinks)
    out.backward(x[3].to(device))
    want = window_cases.expected(*x, window, sinks)
    for name, got in (("out", out), ("dq", q.grad), ("dk", k.grad), ("dv", v.grad)):
        check(got, *want[name], name)
    with torch.no_grad():
        check(ops.sliding_window_attention(q, k, v, window, sinks=sinks), *want["out"])


def test_masks_say_what_they_hold(mojo):
    mask = sliding_window_causal_mask(6, 2, "mojo", sinks=1)
    assert window_and_sinks_of(mask) == (2, 1) and window_of(mask) is None
    plain = sliding_window_causal_mask(6, 2, "mojo")
    assert window_and_sinks_of(plain) == (2, 0) and window_of(plain) == 2
    cpu = sliding_window_causal_mask(6, 2, "cpu", sinks=1)
    assert cpu[5].tolist() == [True, False, False, False, True, True] and torch.equal(mask.cpu(), cpu)
    mask.fill_(True)
    assert window_and_sinks_of(mask) is None


def test_no_rows(device):
    q = torch.zeros(2, 4, 0, 16).to(device)
    assert ops.sliding_window_attention(q, q, q, 3, sinks=1).shape == q.shape


def test_refusals(device):
    q, k, v, _ = (x.to(device) for x in window_cases.inputs(2, 4, 2, 5, 16, torch.float32))
    att = ops.sliding_window_attention
    for kind, call in (
        (ValueError, lambda: att(q, k, v, 0)),
        (ValueError, lambda: att(q, k, v, 3, sinks=-1)),
        (ValueError, lambda: att(q, k, v[:, :, :4], 3)),
        (ValueError, lambda: att(q[:, :, :4], k, v, 3)),
        (ValueError, lambda: att(q[:, :3], k, v, 3)),
        (ValueError, lambda: att(q[0], k[0], v[0], 3)),
        (ValueError, lambda: att(q, k, v, 3, scale=float("nan"))),
        (TypeError, lambda: att(q, k.bfloat16(), v.bfloat16(), 3)),
        (ValueError, lambda: sliding_window_causal_mask(5, 3, device, sinks=-2)),
    ):
        with pytest.raises(kind):
            call()
    if device == "mojo":
        with pytest.raises(TypeError):
            att(q, k.cpu(), v.cpu(), 3)
        with pytest.raises(NotImplementedError):
            att(q.double(), k.double(), v.double(), 3)


@pytest.mark.parametrize("window,sinks", [(3, 0), (3, 2), (30, 0)])
def test_a_gradient_of_the_gradient_is_refused(device, window, sinks):
    """Where it is not known: a second term of a loss must not be left out in silence."""
    x = window_cases.inputs(1, 2, 1, 9, 16, torch.float32)
    q, k, v = (leaf(y, device) for y in x[:3])
    out = ops.sliding_window_attention(q, k, v, window, sinks=sinks)
    dq, = torch.autograd.grad(out.sum(), q, create_graph=True)
    assert dq.requires_grad
    check(dq, *window_cases.expected(*x[:3], torch.ones_like(x[3]), window, sinks)["dq"])
    with pytest.raises(RuntimeError, match="differentia|derivative"):
        (out.sum() + (dq * dq).sum()).backward()


@pytest.mark.parametrize("dtype,d,sinks,new", [(torch.float32, 64, 0, True), (torch.bfloat16, 128, 0, True), (torch.float16, 256, 0, True),
                                               (torch.bfloat16, 96, 0, True), (torch.bfloat16, 64, 0, False), (torch.float16, 64, 0, False),
                                               (torch.bfloat16, 64, 1, True), (torch.float32, 32, 0, True)])
def test_masks_reach_the_windows_kernels(mojo, monkeypatch, dtype, d, sinks, new):
    from torch_mojo_backend.eager_kernels import aten_fast

    if mojo != "host":
        pytest.skip("the stand-in is for machines without a GPU")
    x = [y.to("mojo") for y in window_cases.inputs(1, 2, 1, 9, d, dtype)[:3]]
    mask = sliding_window_causal_mask(9, 3, "mojo", sinks=sinks)
    seen = aten_fast.fused_fa_ex_inputs(*x, mask, 0.0, False, None, True)
    assert seen[3:] == (True, 3, sinks if new else None)
