"""Calls of rotary positions, packed attention and token log-probabilities on the
MI355X whose arguments have to be copied first, or that take kernels of their own."""

import pytest
import torch

import logprob_cases
import packed_cases
from paged_cases import check
from torch_mojo_backend import ops
from torch_mojo_backend.packing import PackedSequences
from torch_mojo_backend.rotary import rotary_frequencies

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _mojo(mojo):
    return mojo


# ---------------------------------------------------------------------------
# copies of arguments live until the call
# ---------------------------------------------------------------------------
def channels_apart(x):
    """x's values in a tensor whose last stride is not 1."""
    return x.transpose(-1, -2).contiguous().to("mojo").transpose(-1, -2)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("which", ["q", "k", "both"])
def test_rotary_of_channels_apart(dtype, which):
    f = rotary_frequencies(32, device="cpu").frequencies
    g = torch.Generator().manual_seed(0)
    x, y = (torch.randn(2, 4, 90, 64, generator=g).to(dtype) for _ in range(2))
    pos = torch.arange(90)
    q = channels_apart(x) if which != "k" else x.to("mojo")
    k = channels_apart(y) if which != "q" else y.to("mojo")
    got = ops.rotary_at(q, k, pos.to("mojo"), f.to("mojo"))
    for name, z, value in (("q", x, got[0]), ("k", y, got[1])):
        check(value, *logprob_cases.turned(z, pos, f, False, 1.0), name)


def test_rotary_of_expanded_gradients():
    f = rotary_frequencies(32, device="cpu").frequencies
    pos = torch.arange(90)
    q, k = (torch.zeros(1, 4, 90, 64).to("mojo").requires_grad_() for _ in range(2))
    a, b = ops.rotary_at(q, k, pos.to("mojo"), f.to("mojo"))
    (2 * a.sum() + 3 * b.sum()).backward()
    for name, value, grad in (("q", 2.0, q.grad), ("k", 3.0, k.grad)):
        check(grad, *logprob_cases.turned(torch.full((1, 4, 90, 64), value), pos, f, False, 1.0, True), name)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_logprobs_of_tokens_apart(dtype):
    """Tokens in a column of a table."""
    x, tokens = logprob_cases.logits(300, 50, dtype)
    pair = torch.stack([tokens, tokens.flip(0)], dim=1).to("mojo")
    d = torch.linspace(-1, 1, 300)
    want = logprob_cases.expected(x, tokens, 0, (d, None, None))
    leaf = x.to("mojo").requires_grad_()
    got = ops.token_logprobs(leaf, pair[:, 0])
    check(got.logprobs, *want["logprobs"])
    got.logprobs.backward(d.to("mojo"))
    check(leaf.grad, *want["dx"])


# ---------------------------------------------------------------------------
# sequences and windows of up to 64 rows, whose backward has bodies of its own
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,d,h,hk", [(BF, 128, 4, 2), (HF, 128, 2, 2), (HF, 120, 2, 1), (HF, 96, 2, 1), (BF, 80, 2, 2), (HF, 64, 2, 1)])
@pytest.mark.parametrize("lengths,window", [([5, 0, 40], 0), ([1], 0), ([300, 64, 1, 65], 64), ([300, 64, 1, 65], 65), ([2] * 20 + [200], 0),
                                            ([64, 65, 63], 0)])
def test_short_and_long_tiles(dtype, d, h, hk, lengths, window):
    """All tiles of one kind or of both, with rows of no sequence around them."""
    at, x = packed_cases.inputs(lengths, h, hk, d, dtype, before=3, behind=9, junk=float("nan"))
    q, k, v = (y.to("mojo").requires_grad_() for y in x[:3])
    out = ops.packed_attention(q, k, v, PackedSequences(torch.tensor(at, dtype=torch.int32).to("mojo"), x[0].shape[0]), window=window)
    out.backward(x[3].to("mojo"))
    want = packed_cases.expected(at, *x, window)
    for name, y in (("out", out), ("dq", q.grad), ("dk", k.grad), ("dv", v.grad)):
        check(y, *want[name], name)
