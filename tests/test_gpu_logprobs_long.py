"""Batches of token log-probabilities that blocks walk a row each, at the lengths
of real vocabularies, on the MI355X against f64."""

import math

import pytest
import torch

from paged_cases import STEP, check
from torch_mojo_backend import ops

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _mojo(mojo):
    return mojo


def expected(x, tokens, d_picked, d_spread):
    """{name: (f64 value, bound)} of rows x.  256 lanes walk a row in batches of 64
    bytes each.  A lane adds a term an element, c / 256 one after another; a batch
    with a new maximum scales its sums, with an exponential and three roundings,
    and its exponents add up to the largest distance from the row's maximum, as does
    the one to the block's; the tree's 10 sums and the settling's 6 roundings
    follow.  A term is off by 2^-22 and its exponent's rounding, |x - m| 2^-23, the
    logarithm by 2^-22 of its value."""
    v = x.double()
    c = v.shape[1]
    z = v - v.amax(-1, keepdim=True)
    e = z.exp()
    s = e.sum(-1, keepdim=True)
    p, ls = e / s, s.log()
    logp = z - ls
    t, t2 = (p * z).sum(-1, keepdim=True), (p * z * z).sum(-1, keepdim=True)
    h = ls - t
    batches = math.ceil(c / (256 * 64 // x.element_size())) + 1
    sums = (math.ceil(c / 256) + 16 + 3 * batches) * 2.0 ** -24 + (2 + batches) * 2.0 ** -22 - z.amin(-1, keepdim=True) * 2.0 ** -23
    e_s = sums + t.abs() * 2.0 ** -23
    ls_err = e_s + 2.0 ** -22 * ls
    h_err = ls_err + (sums + e_s) * t.abs() + t2 * 2.0 ** -23 + 2.0 ** -22 * (ls + t.abs())
    one = torch.zeros_like(v).scatter_(1, tokens[:, None], 1.0)
    g, gh = d_picked.double()[:, None], d_spread.double()[:, None]
    dx = g * one - p * (g + gh * (logp + h))
    part = g.abs() + gh.abs() * (logp.abs() + h)
    rel = (z.abs() + ls) * 2.0 ** -22 + e_s + 2.0 ** -21
    bound = p * ((rel + 4 * 2.0 ** -24) * part + gh.abs() * (logp.abs() * 2.0 ** -21 + h_err))
    bound += 4 * 2.0 ** -24 * (g.abs() * one + dx.abs()) + STEP[x.dtype] * dx.abs() + 2.0 ** -120 * part
    if x.dtype == HF:
        bound += 2.0 ** -25  # half a step of its smallest values
    zt, lt = z.gather(1, tokens[:, None]), logp.gather(1, tokens[:, None])
    lp_err = ls_err + 2.0 ** -23 * (zt.abs() + ls) + 2.0 ** -24 * lt.abs()
    return {"logprobs": (lt[:, 0].numpy(), lp_err[:, 0].numpy()), "entropy": (h[:, 0].numpy(), h_err[:, 0].numpy()),
            "dx": (dx.numpy(), bound.numpy())}


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("n,c", [(512, 50257), (600, 50304), (513, 131071), (520, 262144)])
def test_rows_of_real_vocabularies(dtype, n, c):
    gen = torch.Generator().manual_seed(c)
    x = (3.0 * torch.randn(n, c, generator=gen)).to(dtype)
    tokens = torch.randint(0, c, (n,), generator=gen)
    d_picked, d_spread = torch.randn(n, generator=gen), torch.randn(n, generator=gen)
    rows = [0, 1, 2, 3, 63, 64, 255, 256, 300, n - 2, n - 1]  # (each is walked by itself; some of every alignment)
    want = expected(x[rows], tokens[rows], d_picked[rows], d_spread[rows])
    leaf = x.to("mojo").requires_grad_()
    got = ops.token_logprobs(leaf, tokens.to("mojo"), entropy=True)
    torch.autograd.backward((got.logprobs, got.entropy), (d_picked.to("mojo"), d_spread.to("mojo")))
    dx = torch.stack([leaf.grad[r].cpu() for r in rows])
    for name, y in (("logprobs", got.logprobs.detach().cpu()[rows]), ("entropy", got.entropy.detach().cpu()[rows]), ("dx", dx)):
        check(y, *want[name], name)
    with torch.no_grad():  # (without the entropy, the walk's other kernel)
        check(ops.token_logprobs(leaf, tokens.to("mojo")).logprobs.cpu()[rows], *want["logprobs"])
