"""Rotary positions on the MI355X against f64."""

import pytest
import torch

from logprob_cases import turned
from paged_cases import check
from torch_mojo_backend import ops
from torch_mojo_backend.rotary import rotary_frequencies

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _mojo(mojo):
    return mojo


def rows(b, t, h, d, dtype, seed):
    return torch.randn(b, t, h, d, generator=torch.Generator().manual_seed(seed)).to(dtype).transpose(1, 2)


def run(b, t, h, hk, d, dtype, n, positions, interleaved, scale=1.0, scaling=None, factor=1.0):
    f = rotary_frequencies(n, scaling=scaling, factor=factor, length=512, device="cpu").frequencies
    x = [rows(b, t, m, d, dtype, i) for i, m in enumerate((h, hk, h, hk))]
    q, k = (y.to("mojo").requires_grad_() for y in x[:2])
    got = ops.rotary_at(q, k, positions.to("mojo"), f.to("mojo"), interleaved=interleaved, scale=scale)
    torch.autograd.backward(got, [y.to("mojo") for y in x[2:]])
    for name, y, z in (("q", got[0], x[0]), ("k", got[1], x[1])):
        check(y, *turned(z, positions, f, interleaved, scale), name)
    for name, y, z in (("dq", q.grad, x[2]), ("dk", k.grad, x[3])):
        check(y, *turned(z, positions, f, interleaved, scale, True), name)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("h,hk,d,n", [(4, 1, 256, 256), (2, 2, 64, 32), (3, 1, 96, 96), (1, 1, 80, 40), (2, 1, 20, 10),
                                      (1, 1, 7, 6), (5, 3, 128, 2)])
@pytest.mark.parametrize("b,t", [(1, 1), (2, 37), (1, 300)])
def test_layouts(dtype, interleaved, h, hk, d, n, b, t):
    g = torch.Generator().manual_seed(3)
    run(b, t, h, hk, d, dtype, n, torch.randint(0, 5000, (b, t), generator=g, dtype=torch.int32), interleaved, scale=1.25)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("positions", [torch.arange(70), torch.arange(70, dtype=torch.int32) + 2 ** 31 - 100,
                                       torch.arange(70) - 35, (torch.arange(140) * 1000003).view(2, 70)[:, ::1],
                                       torch.arange(280, dtype=torch.int32).view(2, 140)[:, ::2]])
def test_positions(dtype, positions):
    run(2, 70, 2, 1, 64, dtype, 64, positions, False)


@pytest.mark.parametrize("scaling", ["linear", "base", "parts"])
def test_scalings(scaling):
    run(1, 50, 2, 1, 64, F32, 64, torch.arange(50) * 997, True, scaling=scaling, factor=8.0)


def test_packed_rows_and_one_side():
    f = rotary_frequencies(64, device="cpu").frequencies
    x = rows(1, 90, 3, 64, BF, 0)[0].transpose(0, 1)  # [tokens, heads, d]
    pos = torch.randint(0, 90, (90,), dtype=torch.int32)
    q, k = ops.rotary_at(x.to("mojo"), None, pos.to("mojo"), f.to("mojo"))
    assert k is None
    want = turned(x.transpose(0, 1)[None], pos, f, False, 1.0)
    check(q, *(y[0].swapaxes(0, 1) for y in want))
    q, k = ops.rotary_at(None, x.to("mojo"), pos.to("mojo"), f.to("mojo"))
    assert q is None
    check(k, *(y[0].swapaxes(0, 1) for y in want))
    leaf = x.to("mojo").requires_grad_()
    q, k = ops.rotary_at(leaf, x.to("mojo"), pos.to("mojo"), f.to("mojo"))
    k.sum()
    q.sum().backward()
    check(leaf.grad, *(y[0].swapaxes(0, 1) for y in turned(torch.ones_like(x).transpose(0, 1)[None], pos, f, False, 1.0, True)))


def test_strides():
    """Slices of a projection, rows at odd offsets, heads first, repeated rows."""
    f = rotary_frequencies(32, device="cpu").frequencies
    fm, pos = f.to("mojo"), torch.arange(40, dtype=torch.int32)
    x = rows(2, 40, 2, 64, BF, 5)
    want = turned(x, pos, f, False, 1.0)
    wide = torch.zeros(2, 2, 40, 65, dtype=BF)
    wide[..., 1:] = x
    both = torch.cat([x, x], dim=-1)
    one = x[:, :1].expand(2, 3, 40, 64)
    pm = pos.to("mojo")
    for y in (wide.to("mojo")[..., 1:], both.to("mojo")[..., 64:], x.contiguous().to("mojo")):
        check(ops.rotary_at(y, None, pm, fm)[0], *want)
    check(ops.rotary_at(x[:, :1].to("mojo").expand(2, 3, 40, 64), None, pm, fm)[0], *turned(one, pos, f, False, 1.0))
    flipped = ops.rotary_at(x.transpose(-1, -2).contiguous().to("mojo").transpose(-1, -2), None, pm, fm)[0]
    check(flipped, *want)


def test_many_rows():
    run(3, 2000, 8, 2, 128, BF, 128, torch.arange(2000), False)


def test_nothing_is_turned_or_there():
    f = torch.zeros(0, dtype=torch.float64)
    x = rows(1, 5, 2, 16, BF, 0)
    got = ops.rotary_at(x.to("mojo"), None, torch.arange(5).to("mojo"), f.to("mojo"))[0]
    assert torch.equal(got.cpu(), x)
    none = torch.zeros(2, 3, 0, 16, dtype=BF).to("mojo")
    assert ops.rotary_at(none, none, torch.zeros(0, dtype=torch.int64).to("mojo"), f.to("mojo"))[0].shape == none.shape


def test_gradient_of_the_gradient():
    """The map is linear: its gradient's gradient is the map again."""
    f = rotary_frequencies(16, device="cpu").frequencies
    pos = torch.arange(6)
    x, dy, w = (rows(1, 6, 2, 16, F32, i) for i in range(3))
    q = x.to("mojo").requires_grad_()
    g = dy.to("mojo").requires_grad_()
    out = ops.rotary_at(q, None, pos.to("mojo"), f.to("mojo"))[0]
    dx, = torch.autograd.grad(out, q, g, create_graph=True)
    back, = torch.autograd.grad(dx, g, w.to("mojo"))
    check(back, *turned(w, pos, f, False, 1.0))
