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
