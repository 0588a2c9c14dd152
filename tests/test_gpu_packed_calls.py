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


# ---------------------------------------------------------------------------
# what autograd sees
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [HF, F32])
def test_saved_tensors_through_a_hook(dtype):
    """From copies on the host, given back dense or every second element of a wider tensor."""
    at, x = packed_cases.inputs([70, 0, 9], 4, 2, 64, dtype, behind=2)
    want = packed_cases.expected(at, *x)
    logits, tokens = logprob_cases.logits(6, 400, dtype)
    ones = [torch.ones(6), torch.ones(6), torch.ones(6, 3)]
    dx = logprob_cases.expected(logits, tokens, 3, ones)["dx"]
    seqs = PackedSequences(torch.tensor(at, dtype=torch.int32).to("mojo"), x[0].shape[0])
    for give in (lambda t: t.to("mojo"), lambda t: torch.stack([t, t], dim=-1).to("mojo")[..., 0]):
        q, k, v = (y.to("mojo").requires_grad_() for y in x[:3])
        leaf = logits.to("mojo").requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), give):
            out = ops.packed_attention(q, k, v, seqs)
            got = ops.token_logprobs(leaf, tokens.to("mojo"), top=3, entropy=True)
        out.backward(x[3].to("mojo"))
        for name, y in (("out", out), ("dq", q.grad), ("dk", k.grad), ("dv", v.grad)):
            check(y, *want[name], name)
        torch.autograd.backward(got[:3], [y.to("mojo") for y in ones])
        check(leaf.grad, *dx, "dx")


def test_tangents_are_refused():
    from torch.autograd import forward_ad as fwd

    f = rotary_frequencies(64, device="cpu").frequencies.to("mojo")
    x = torch.randn(9, 2, 64).to("mojo")
    seqs = PackedSequences.of_lengths([5, 4])
    with fwd.dual_level():
        dual = fwd.make_dual(x, x.clone())
        for call in (lambda: ops.packed_attention(x, dual, x, seqs), lambda: ops.rotary_at(dual, None, seqs.positions, f),
                     lambda: ops.token_logprobs(dual, entropy=True)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_gradients_of_no_rows():
    seqs = PackedSequences.of_lengths([0, 0])
    q, k, v = (torch.zeros(0, h, 64).to("mojo").requires_grad_() for h in (4, 2, 2))
    ops.packed_attention(q, k, v, seqs).sum().backward()
    assert [tuple(y.grad.shape) for y in (q, k, v)] == [(0, 4, 64), (0, 2, 64), (0, 2, 64)]


def test_workspace_of_an_unsplit_backward():
    """A grouped backward without partials takes no more memory than its results and row terms."""
    t, h, hk, d = 8192, 32, 8, 128
    x = [torch.zeros(t, n, d, dtype=BF).to("mojo").requires_grad_() for n in (h, hk, hk)]
    dy = torch.zeros(t, h, d, dtype=BF).to("mojo")
    out = ops.packed_attention(*x, PackedSequences.of_lengths([t]))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out.backward(dy)
    torch.cuda.synchronize()
    results, terms = 2 * t * (h + 2 * hk) * d, 2 * 4 * t * h
    assert results <= torch.cuda.max_memory_allocated() - before <= results + terms + (4 << 20)  # (blocks of 2 MB)
