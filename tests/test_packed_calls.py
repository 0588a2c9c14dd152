"""Calls of rotary positions, packed attention and token log-probabilities whose
arguments have to be copied first, or that autograd has to know of, off the GPU."""

import pytest
import torch

import logprob_cases
import packed_standin  # noqa: F401
from paged_cases import check
from torch_mojo_backend import ops
from torch_mojo_backend.rotary import rotary_frequencies

F32 = torch.float32


@pytest.fixture
def device(mojo):
    if mojo != "host":
        pytest.skip("the stand-in is for machines without a GPU")
    return "mojo"


# ---------------------------------------------------------------------------
# copies of arguments live until the call
# ---------------------------------------------------------------------------
def channels_apart(x):
    """x's values in a tensor whose last stride is not 1."""
    return x.transpose(-1, -2).contiguous().to("mojo").transpose(-1, -2)


@pytest.mark.parametrize("which", ["q", "k", "both"])
def test_rotary_of_channels_apart(device, which):
    f = rotary_frequencies(32, device="cpu").frequencies
    g = torch.Generator().manual_seed(0)
    x, y = (torch.randn(2, 4, 90, 64, generator=g) for _ in range(2))
    pos = torch.arange(90)
    q = channels_apart(x) if which != "k" else x.to("mojo")
    k = channels_apart(y) if which != "q" else y.to("mojo")
    got = ops.rotary_at(q, k, pos.to("mojo"), f.to("mojo"))
    for name, z, value in (("q", x, got[0]), ("k", y, got[1])):
        check(value, *logprob_cases.turned(z, pos, f, False, 1.0), name)


def test_rotary_of_expanded_gradients(device):
    f = rotary_frequencies(32, device="cpu").frequencies
    pos = torch.arange(90)
    q, k = (torch.zeros(1, 4, 90, 64).to("mojo").requires_grad_() for _ in range(2))
    a, b = ops.rotary_at(q, k, pos.to("mojo"), f.to("mojo"))
    (2 * a.sum() + 3 * b.sum()).backward()
    for name, value, grad in (("q", 2.0, q.grad), ("k", 3.0, k.grad)):
        check(grad, *logprob_cases.turned(torch.full((1, 4, 90, 64), value), pos, f, False, 1.0, True), name)


@pytest.mark.parametrize("entropy", [False, True])
def test_logprobs_of_tokens_apart(device, monkeypatch, entropy):
    """Tokens in a column of a table, also by the first call that may raise at a host read."""
    from torch_mojo_backend.eager_kernels import aten_fast

    x, tokens = logprob_cases.logits(300, 50, F32)
    pair = torch.stack([tokens, tokens.flip(0)], dim=1).to("mojo")
    d = torch.linspace(-1, 1, 300)
    want = logprob_cases.expected(x, tokens, 0, (d, None, None))
    for flags in (aten_fast._error_flags, {}):
        monkeypatch.setattr(aten_fast, "_error_flags", flags)
        leaf = x.to("mojo").requires_grad_()
        got = ops.token_logprobs(leaf, pair[:, 0], entropy=entropy)
        check(got.logprobs, *want["logprobs"])
        got.logprobs.backward(d.to("mojo"))
        check(leaf.grad, *want["dx"])
