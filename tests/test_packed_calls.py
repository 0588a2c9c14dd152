"""Calls of rotary positions, packed attention and token log-probabilities whose
arguments have to be copied first, or that autograd has to know of, off the GPU."""

import pytest
import torch

import decode_cases
import logprob_cases
import packed_cases
import packed_standin  # noqa: F401
from host_standin import HostStandIn
from paged_cases import check
from torch_mojo_backend import ops
from torch_mojo_backend.packing import PackedSequences
from torch_mojo_backend.rotary import rotary_frequencies

BF, F32 = torch.bfloat16, torch.float32

HostStandIn.mi355x_packed_attn_bwd_workspace_bytes_for = lambda self, *a: 64


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


def test_cross_entropy_of_targets_apart(device):
    x, tokens = logprob_cases.logits(300, 50, F32)
    pair = torch.stack([tokens, tokens.flip(0)], dim=1)
    want, leaf = (y.requires_grad_() for y in (x.clone(), x.to("mojo")))
    for y, t in ((want, pair), (leaf, pair.to("mojo"))):
        torch.nn.functional.cross_entropy(y, t[:, 0], reduction="none").sum().backward()
    assert torch.allclose(leaf.grad.cpu(), want.grad, rtol=0, atol=1e-6)  # (both f32, of values up to 1)


# ---------------------------------------------------------------------------
# what a backward keeps is autograd's
# ---------------------------------------------------------------------------
def saved_by(call, give=lambda t: t.to("mojo")):
    """The call's result, and the tensors that a saved-tensor hook sees of it, in
    whose places the backward gets others of the same values."""
    seen = []

    def pack(t):
        seen.append((tuple(t.shape), t.dtype))
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, give):
        out = call()
    return out, seen


def test_saved_tensors_of_attention(device):
    at, x = packed_cases.inputs([5, 0, 9], 4, 2, 16, BF, behind=2)
    seqs = PackedSequences(torch.tensor(at, dtype=torch.int32).to("mojo"), 16)
    q, k, v = (y.to("mojo").requires_grad_() for y in x[:3])
    out, seen = saved_by(lambda: ops.packed_attention(q, k, v, seqs))
    rows, kv = ((16, 4, 16), BF), ((16, 2, 16), BF)
    assert sorted(seen, key=str) == sorted([rows, kv, kv, rows, ((4, 16), F32), rows], key=str)
    out.backward(x[3].to("mojo"))
    want = packed_cases.expected(at, *x)
    for name, y in (("out", out), ("dq", q.grad), ("dk", k.grad), ("dv", v.grad)):
        check(y, *want[name], name)


def test_saved_tensors_of_logprobs(device):
    x, tokens = logprob_cases.logits(6, 40, F32)
    leaf = x.to("mojo").requires_grad_()
    got, seen = saved_by(lambda: ops.token_logprobs(leaf, tokens.to("mojo"), top=3, entropy=True))
    assert ((6, 2), F32) in seen and len(seen) == 5
    ones = [torch.ones(6), torch.ones(6), torch.ones(6, 3)]
    torch.autograd.backward(got[:3], [y.to("mojo") for y in ones])
    check(leaf.grad, *logprob_cases.expected(x, tokens, 3, ones)["dx"])


def test_saved_tensors_come_back_apart(device):
    """From a hook that gives back every second element of a wider tensor."""
    def apart(t):
        return torch.stack([t, t], dim=-1).to("mojo")[..., 0]

    at, x = packed_cases.inputs([5, 9], 4, 2, 16, BF)
    seqs = PackedSequences(torch.tensor(at, dtype=torch.int32).to("mojo"), 14)
    q, k, v = (y.to("mojo").requires_grad_() for y in x[:3])
    saved_by(lambda: ops.packed_attention(q, k, v, seqs), apart)[0].backward(x[3].to("mojo"))
    want = packed_cases.expected(at, *x)
    for name, y in (("dq", q.grad), ("dk", k.grad), ("dv", v.grad)):
        check(y, *want[name], name)
    x, tokens = logprob_cases.logits(6, 40, F32)
    leaf = x.to("mojo").requires_grad_()
    got, _ = saved_by(lambda: ops.token_logprobs(leaf, tokens.to("mojo"), top=3, entropy=True), apart)
    ones = [torch.ones(6), torch.ones(6), torch.ones(6, 3)]
    torch.autograd.backward(got[:3], [y.to("mojo") for y in ones])
    check(leaf.grad, *logprob_cases.expected(x, tokens, 3, ones)["dx"])


def test_nothing_is_kept_behind_a_backward(device):
    """A loss that a program keeps holds none of what the backward read."""
    at, x = packed_cases.inputs([5, 9], 2, 2, 16, BF)
    seqs = PackedSequences(torch.tensor(at, dtype=torch.int32).to("mojo"), 14)
    out = ops.packed_attention(*(y.to("mojo").requires_grad_() for y in x[:3]), seqs)
    logits, tokens = logprob_cases.logits(6, 40, F32)
    lp = ops.token_logprobs(logits.to("mojo").requires_grad_(), tokens.to("mojo")).logprobs
    for y in (out, lp):
        node = y.grad_fn
        y.sum().backward()
        held = [z for z in vars(node).values() for z in (z if isinstance(z, tuple) else (z,)) if isinstance(z, torch.Tensor)]
        assert not held, [tuple(z.shape) for z in held]
        with pytest.raises(RuntimeError, match="second time"):
            node.saved_tensors


# ---------------------------------------------------------------------------
# tangents
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(device, grad):
    """No operator has a forward-mode derivative: a dual tensor is refused, not taken as a constant."""
    from torch.autograd import forward_ad as fwd

    at, x = packed_cases.inputs([5, 9], 2, 2, 16, F32)
    seqs = PackedSequences(torch.tensor(at, dtype=torch.int32).to("mojo"), 14)
    q, k, v, t = (y.to("mojo") for y in x)
    logits, tokens = (y.to("mojo") for y in logprob_cases.logits(14, 32, F32))
    f, pos = rotary_frequencies(16, device="cpu").frequencies.to("mojo"), seqs.positions
    if grad:
        for y in (q, k, v, logits):
            y.requires_grad_()
    with fwd.dual_level():
        dual = fwd.make_dual(q, t)
        wide = fwd.make_dual(logits, t.reshape(14, 32))
        for call in (
            lambda: ops.packed_attention(dual, k, v, seqs),
            lambda: ops.packed_attention(q, dual, v, seqs, window=3, scale=0.5),
            lambda: ops.packed_attention(q, k, dual, seqs),
            lambda: ops.rotary_at(dual, k, pos, f),
            lambda: ops.rotary_at(q, dual, pos, f, scale=2),
            lambda: ops.rotary_at(None, dual, pos, f),
            lambda: ops.token_logprobs(wide, tokens),
            lambda: ops.token_logprobs(wide.view(2, 7, 32), top=2),
        ):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        if grad:  # nor have the backward passes
            lp = ops.token_logprobs(logits, tokens).logprobs
            for out, at, g in ((ops.packed_attention(q, k, v, seqs), q, t), (ops.rotary_at(q, None, pos, f)[0], q, t),
                               (lp, logits, t[:, 0, 0])):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    torch.autograd.grad(out, at, fwd.make_dual(g.clone(), g.clone()))
        assert ops.packed_attention(q, k, v, seqs).shape == (14, 2, 16)  # none of its inputs has a tangent
        assert ops.rotary_at(q, k, pos, f)[0].shape == q.shape
    assert ops.token_logprobs(logits, tokens).logprobs.shape == (14,)


# ---------------------------------------------------------------------------
# a model that has answered before it trains
# ---------------------------------------------------------------------------
def test_training_after_inference(device):
    m, ref = decode_cases.model(F32, "mojo", sinks=0)
    idx = torch.randint(0, 97, (12,), generator=torch.Generator().manual_seed(2)).to("mojo")
    with torch.inference_mode():
        m.forward_packed(idx, PackedSequences.of_lengths([5, 7]))
    m.score_packed(idx, PackedSequences.of_lengths([5, 7])).logprobs.sum().backward()
    ref.score_packed(idx.cpu(), PackedSequences.of_lengths([5, 7], device="cpu")).logprobs.sum().backward()
    for (name, p), r in zip(m.named_parameters(), ref.parameters()):
        check(p.grad, r.grad.numpy(), 2e-5 * max(1.0, r.grad.abs().max().item()) + 0 * r.grad.numpy(), name)


@pytest.mark.parametrize("at,tokens", [([0], 0), ([3], 5), ([0, 0, 0], 0)])
@pytest.mark.parametrize("where", ["cpu", "mojo"])
def test_gradients_of_no_rows(device, where, at, tokens):
    """Zeros for each of q, k and v, whichever of them takes one."""
    seqs = PackedSequences(torch.tensor(at, dtype=torch.int32).to(where), tokens)
    for some in ((0, 1, 2), (1,), (2,)):
        x = [torch.full((tokens, h, 16), float("nan")).to(where) for h in (4, 2, 2)]
        for i in some:
            x[i].requires_grad_()
        out = ops.packed_attention(*x, seqs)
        out.sum().backward()
        assert out.shape == (tokens, 4, 16) and not out.detach().cpu().any()
        for i in some:
            assert x[i].grad.shape == x[i].shape and not x[i].grad.cpu().any()


def test_no_channels(device):
    for where in ("cpu", "mojo"):
        q, k = torch.zeros(5, 4, 0).to(where), torch.zeros(5, 2, 0).to(where).requires_grad_()
        out = ops.packed_attention(q, k, k, PackedSequences.of_lengths([5], device=where))
        out.sum().backward()
        assert out.shape == q.shape and k.grad.shape == k.shape
