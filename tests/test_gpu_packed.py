"""Attention over packed sequences on the MI355X against f64, forward and
backward, over types, head layouts, lengths and what lies between and behind
the sequences."""

import itertools

import pytest
import torch

import packed_cases as cases
from paged_cases import check
from torch_mojo_backend import ops
from torch_mojo_backend.packing import PackedSequences

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _mojo(mojo):
    return mojo


def sequences(at, tokens):
    return PackedSequences(torch.tensor(at, dtype=torch.int32).to("mojo"), tokens)


def run(at, x, window=0, scale=None):
    seqs = sequences(at, x[0].shape[0])
    q, k, v = (y.to("mojo").requires_grad_() for y in x[:3])
    out = ops.packed_attention(q, k, v, seqs, window=window, scale=scale)
    out.backward(x[3].to("mojo"))
    return {"out": out, "dq": q.grad, "dk": k.grad, "dv": v.grad}


def compare(got, want):
    for name, value in got.items():
        check(value, *want[name], name)


LENGTHS = [[1], [2], [64], [65, 1, 127], [128, 129], [0, 5, 0, 0, 300, 1, 0], [1] * 70, [200, 333], [31, 97, 256, 3]]


@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("before,behind", [(0, 0), (3, 140)])
def test_positions(lengths, before, behind):
    at = [before, *(before + n for n in itertools.accumulate(lengths))]
    tokens = at[-1] + behind
    got = sequences(at, tokens).positions.cpu()
    want = torch.zeros(tokens, dtype=torch.int32)
    for a, b in itertools.pairwise(at):
        want[a:b] = torch.arange(b - a)
    assert torch.equal(got, want)


def test_positions_of_many_and_of_long_sequences():
    for lengths in ([1] * 5000, [3, 0, 1] * 700, [100000, 1, 70000], [64, 65] * 300):
        at = [0, *itertools.accumulate(lengths)]
        got = sequences(at, at[-1]).positions.cpu()
        assert torch.equal(got, torch.cat([torch.arange(n) for n in lengths]).int())


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("d,h,hk", [(64, 2, 2), (128, 4, 1), (256, 4, 2)])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_forward_and_backward(dtype, d, h, hk, lengths):
    at, x = cases.inputs(lengths, h, hk, d, dtype)
    compare(run(at, x), cases.expected(at, *x))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d,h,hk", [(8, 1, 1), (40, 3, 1), (72, 2, 2), (88, 2, 1), (96, 4, 2), (112, 2, 2), (136, 2, 1), (160, 3, 3),
                                    (192, 4, 2), (200, 2, 1), (248, 2, 2)])
def test_other_head_dims(dtype, d, h, hk):
    at, x = cases.inputs([70, 0, 1, 190, 64], h, hk, d, dtype, before=2, behind=70)
    compare(run(at, x), cases.expected(at, *x))


@pytest.mark.parametrize("dtype,d,h,hk", [(BF, 64, 2, 2), (BF, 128, 4, 2), (HF, 256, 2, 1), (BF, 96, 2, 1), (BF, 192, 2, 2),
                                         (F32, 64, 2, 1), (F32, 256, 1, 1)])
@pytest.mark.parametrize("window", [1, 17, 64, 100, 128, 2 ** 40])
def test_windows(dtype, d, h, hk, window):
    at, x = cases.inputs([300, 1, 64, 190], h, hk, d, dtype, behind=9)
    compare(run(at, x, window), cases.expected(at, *x, min(window, 1000)))


@pytest.mark.parametrize("dtype,d", [(BF, 64), (HF, 128), (BF, 256), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.0, 1e-30])
def test_scales(dtype, d, scale):
    at, x = cases.inputs([130, 77], 2, 1, d, dtype)
    compare(run(at, x, 0, scale), cases.expected(at, *x, 0, scale))


@pytest.mark.parametrize("dtype,d,h,hk", [(BF, 64, 12, 12), (BF, 128, 8, 2), (BF, 256, 4, 1), (F32, 64, 2, 2)])
def test_long_sequences(dtype, d, h, hk):
    at, x = cases.inputs([1500, 3, 700], h, hk, d, dtype, behind=1)
    compare(run(at, x), cases.expected(at, *x))


@pytest.mark.parametrize("dtype,d,h,hk,window", [(BF, 256, 32, 4, 0), (HF, 192, 32, 32, 0), (BF, 160, 32, 2, 100), (BF, 256, 32, 32, 65),
                                                 (BF, 96, 32, 8, 0)])
def test_many_blocks(dtype, d, h, hk, window):
    at, x = cases.inputs([300, 1, 0, 260, 700, 128, 64, 127, 500], h, hk, d, dtype, behind=30)
    compare(run(at, x, window), cases.expected(at, *x, window))


def test_nothing_reaches_another_sequence_of_many_blocks():
    lengths, h, d = [300, 700, 1100], 32, 192
    at, x = cases.inputs(lengths, h, 4, d, BF, behind=60, junk=float("nan"))
    want = cases.expected(at, *x)
    for y, value in zip(x, (float("inf"), float("nan"), float("-inf"), float("nan"))):
        y[at[1] + 3:at[2]:4] = value
    got = {n: y.detach().cpu() for n, y in run(at, x).items()}
    for name, y in got.items():
        for a, b in ((0, at[1]), (at[2], x[0].shape[0])):
            check(y[a:b], *(z[a:b] for z in want[name]), name)


@pytest.mark.parametrize("dtype,d", [(BF, 64), (BF, 128), (HF, 256), (F32, 64), (BF, 96), (F32, 96), (BF, 192), (HF, 160)])
def test_nothing_reaches_another_sequence(dtype, d):
    """NaN and infinities in the rows of no sequence and in one of three sequences."""
    lengths = [45, 30, 81]
    at, x = cases.inputs(lengths, 2, 1, d, dtype, before=7, behind=60, junk=float("nan"))
    want = cases.expected(at, *x)
    for y, value in zip(x, (float("inf"), float("nan"), float("-inf"), float("nan"))):
        y[at[1] + 3:at[2]:4] = value
    got = {n: y.detach().cpu() for n, y in run(at, x).items()}
    for name, y in got.items():
        for a, b in ((0, at[1]), (at[2], x[0].shape[0])):
            check(y[a:b], *(z[a:b] for z in want[name]), name)


@pytest.mark.parametrize("dtype,d", [(BF, 64), (HF, 128), (F32, 64), (BF, 40)])
def test_strides_and_alignment(dtype, d):
    """Rows of one packed projection, rows at odd offsets, heads first, a row that is repeated, and an expanded gradient."""
    h = 2
    at, x = cases.inputs([100, 51], h, h, d, dtype)
    want = cases.expected(at, *x)
    t = x[0].shape[0]
    whole = torch.cat([y.reshape(t, h * d) for y in x[:3]], dim=-1).to("mojo").requires_grad_()
    out = ops.packed_attention(*(y.view(t, h, d) for y in whole.split(h * d, dim=-1)), sequences(at, t))
    out.backward(x[3].to("mojo"))
    got = [y.reshape(t, h, d) for y in whole.grad.cpu().split(h * d, dim=-1)]
    compare(dict(zip(("out", "dq", "dk", "dv"), (out, *got))), want)

    def odd(y):
        wide = torch.zeros(t, h, d + 1, dtype=dtype)
        wide[..., 1:] = y
        return wide.to("mojo")[..., 1:]

    first = [y.transpose(0, 1).contiguous().to("mojo").transpose(0, 1) for y in x[:3]]
    for q, k, v in ([odd(y) for y in x[:3]], first):
        with torch.no_grad():
            check(ops.packed_attention(q, k, v, sequences(at, t)), *want["out"])
    one = x[1][:1].expand(t, h, d)
    ones = torch.ones(1, 1, 1, dtype=dtype).expand(t, h, d)
    want = cases.expected(at, x[0], one, x[2], ones)
    q, k, v = (y.to("mojo").requires_grad_() for y in (x[0], x[1][:1], x[2]))
    ops.packed_attention(q, k.expand(t, h, d), v, sequences(at, t)).backward(torch.ones(1, 1, 1, dtype=dtype).to("mojo").expand(t, h, d))
    check(q.grad, *want["dq"])
    check(v.grad, *want["dv"])


def test_one_tensor_as_all_three():
    at, (x, _, _, dy) = cases.inputs([90, 40], 2, 2, 64, F32)
    leaf = x.to("mojo").requires_grad_()
    ops.packed_attention(leaf, leaf, leaf, sequences(at, 130)).backward(dy.to("mojo"))
    want = cases.expected(at, x, x, x, dy)
    check(leaf.grad, sum(want[n][0] for n in ("dq", "dk", "dv")), sum(want[n][1] for n in ("dq", "dk", "dv")) + 2.0 ** -20)


def test_results_repeat():
    at, x = cases.inputs([300, 20, 700], 4, 2, 128, BF)
    a, b = run(at, x), run(at, x)
    for n in a:
        assert torch.equal(a[n].detach().cpu(), b[n].detach().cpu()), n


@pytest.mark.parametrize("offsets", [[0, 5, 4, 9], [-1, 5], [0, 11], [5, 3], [0, 2 ** 31 - 1]])
def test_bad_offsets_raise_and_leave_zeros(offsets):
    _, x = cases.inputs([10], 2, 1, 64, BF)
    seqs = sequences(offsets, 10)
    with torch.no_grad():
        out = ops.packed_attention(*(y.to("mojo") for y in x[:3]), seqs)
    with pytest.raises(IndexError, match="packed sequences"):
        out.cpu()
    assert not out.cpu().float().abs().any() and not seqs.positions.cpu().any()


def test_only_padding():
    _, x = cases.inputs([], 2, 1, 64, F32, behind=100, junk=float("nan"))
    got = run([0], x)
    assert all(not y.detach().cpu().abs().any() for y in got.values())


def test_one_tensor_for_all_and_gradients_of_some():
    at, x = cases.inputs([70, 1, 100], 2, 2, 64, BF)
    seqs = sequences(at, 171)
    want = cases.expected(at, x[0], x[0], x[0], x[3])
    leaf = x[0].to("mojo").requires_grad_()
    ops.packed_attention(leaf, leaf, leaf, seqs).backward(x[3].to("mojo"))
    value = sum(want[n][0] for n in ("dq", "dk", "dv"))
    # (each rounded, and two sums of them)
    bound = sum(want[n][1] for n in ("dq", "dk", "dv")) + 2.0 ** -8 * (abs(value) + abs(want["dq"][0] + want["dk"][0]) + abs(want["dk"][0] + want["dv"][0]))
    check(leaf.grad, value, bound)
    want = cases.expected(at, *x)
    q, k, v = (y.to("mojo") for y in x[:3])
    k.requires_grad_()
    out = ops.packed_attention(q, k, v, seqs)
    for _ in range(2):  # the graph is kept
        dk, = torch.autograd.grad(out, k, x[3].to("mojo"), retain_graph=True)
        check(dk, *want["dk"])
    with torch.no_grad():
        out.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, k, x[3].to("mojo"))


def test_leaves_of_one_buffer_keep_their_gradients():
    at, x = cases.inputs([40, 30], 2, 2, 64, F32)
    whole = torch.cat(x[:3], dim=1).to("mojo")
    q, k, v = (y.detach().requires_grad_() for y in whole.split(2, dim=1))
    ops.packed_attention(q, k, v, sequences(at, 70)).backward(x[3].to("mojo"))
    before = k.grad.clone()
    torch.cat([q.grad, k.grad, v.grad], dim=1).mul_(3)
    assert torch.equal(before.cpu(), k.grad.cpu())
    check(k.grad, *cases.expected(at, *x)["dk"])


def test_many_short_sequences_and_far_rows():
    """As many tiles as rows, and rows that lie further apart than the kernels' offsets reach."""
    n, h, d = 30000, 2, 8
    at, x = cases.inputs([1] * n, h, 1, d, BF)
    got = run(at, x)
    assert torch.equal(got["out"].cpu(), x[2].expand(n, h, d))  # a row that sees itself
    # dS = P (dP - D) is 0 but for dP and D, the same 8 products added in f32 in two
    # orders: 8 roundings each, and their difference's and the next product's
    q, k, v, dy = (y.double() for y in x)
    off = d ** -0.5 * 20 * 2.0 ** -24 * (dy * v).abs().sum(-1, keepdim=True)
    assert (got["dq"].cpu().double().abs() <= off * k.abs()).all()
    assert (got["dk"].cpu().double().abs() <= (off * q.abs()).sum(1, keepdim=True)).all()
    check(got["dv"], x[3].double().sum(1, keepdim=True).numpy(), 2.0 ** -8 * x[3].double().sum(1, keepdim=True).abs().numpy() + 2.0 ** -22)
    at, x = cases.inputs([5, 3], 1, 1, 64, BF)
    far = torch.zeros(8, 2 ** 25 + 64, dtype=BF, device="mojo")
    far[:, :64] = x[1].view(8, 64).to("mojo")
    k = far[:, :64].view(8, 1, 64)
    with torch.no_grad():
        check(ops.packed_attention(x[0].to("mojo"), k, x[2].to("mojo"), sequences(at, 8)), *cases.expected(at, *x)["out"])


def test_no_sequences():
    at, x = cases.inputs([], 2, 1, 64, BF, behind=70)
    for y in run(at, x).values():
        assert not y.detach().cpu().any()


@pytest.mark.parametrize("dtype,d,h,hk", [(BF, 64, 12, 12), (HF, 64, 12, 12), (BF, 128, 8, 2), (BF, 80, 8, 8), (BF, 256, 4, 4)])
@pytest.mark.parametrize("lengths", [[2] * 40, [2, 3, 5, 7, 9] * 8])
def test_gradients_of_few_terms(dtype, d, h, hk, lengths):
    """The norm of what dQ and dK of short sequences are off by: that of rounding them,
    whose error is spread evenly over half a step to either side, a root of three of
    half a step at most.  (dS rounded once would add as much again.)"""
    at, x = cases.inputs(lengths, h, hk, d, dtype)
    got, want = run(at, x), cases.expected(at, *x)
    for name in ("dq", "dk"):
        value = torch.from_numpy(want[name][0])
        off = (got[name].cpu().double() - value).norm() / value.norm()
        assert off <= torch.finfo(dtype).eps / 2 / 3 ** 0.5, (name, off.item())
