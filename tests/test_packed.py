"""Packed sequences, rotary positions and token log-probabilities off the GPU:
against f64, the models that use them, and refusals."""

import itertools
import math

import numpy as np
import pytest
import torch

import decode_cases
import logprob_cases
import packed_cases as cases
import packed_standin  # noqa: F401
import paged_standin  # noqa: F401
from paged_cases import check
from torch_mojo_backend import ops
from torch_mojo_backend.gemma3 import Gemma3, Gemma3Config
from torch_mojo_backend.gpt2 import GPT, GPTConfig, training_step
from torch_mojo_backend.packing import PackedSequences
from torch_mojo_backend.rotary import rotary_frequencies

F32 = torch.float32


@pytest.fixture(params=["cpu", "mojo"])
def device(request, mojo):
    if request.param == "mojo" and mojo != "host":
        pytest.skip("the stand-in is for machines without a GPU")
    return request.param


def offsets(at, device):
    return torch.tensor(at, dtype=torch.int32).to(device)


@pytest.mark.parametrize("lengths,before,behind", [([3, 0, 4], 0, 0), ([1], 2, 3), ([], 0, 5), ([5, 1, 1, 2], 1, 0), ([], 0, 0)])
@pytest.mark.parametrize("window", [0, 2])
def test_attention(device, lengths, before, behind, window):
    at, x = cases.inputs(lengths, 4, 2, 16, F32, before=before, behind=behind, junk=float("nan") if lengths else 0.0)
    seqs = PackedSequences(offsets(at, device), x[0].shape[0])
    q, k, v = (y.to(device).requires_grad_() for y in x[:3])
    out = ops.packed_attention(q, k, v, seqs, window=window)
    out.backward(x[3].to(device))
    want = cases.expected(at, *x, window)
    got = {"out": out, "dq": q.grad, "dk": k.grad, "dv": v.grad}
    for name, value in got.items():
        check(value if value is not None else torch.zeros_like(q if name == "dq" else k), *want[name], name)
    with torch.no_grad():
        check(ops.packed_attention(q, k, v, seqs, window=window), *want["out"])


def test_sequences(device):
    seqs = PackedSequences.of_lengths([2, 0, 3], 7, device=device)
    assert seqs.positions.cpu().tolist() == [0, 1, 0, 1, 2, 0, 0] and seqs.count == 3
    ids = torch.arange(10, 17).to(device)
    assert seqs.next_tokens(ids).cpu().tolist() == [11, -100, 13, 14, -100, -100, -100]
    assert PackedSequences.of_lengths([], device=device).positions.shape == (0,)
    empty = PackedSequences.of_lengths([0, 0], device=device)
    assert empty.next_tokens(torch.zeros(0, dtype=torch.int64).to(device)).shape == (0,)
    for kind, call in (
        (ValueError, lambda: PackedSequences(offsets([0, 3], device).long(), 3)),
        (ValueError, lambda: PackedSequences(offsets([[0, 3]], device), 3)),
        (ValueError, lambda: PackedSequences(offsets([], device), 3)),
        (ValueError, lambda: PackedSequences(offsets([0, 3], device), -1)),
        (ValueError, lambda: PackedSequences(offsets([0, 3], device), 2 ** 30)),
        (ValueError, lambda: PackedSequences.of_lengths([3, -1], device=device)),
        (ValueError, lambda: PackedSequences.of_lengths([3, 4], 6, device=device)),
        (ValueError, lambda: PackedSequences.of_lengths([2 ** 30], device=device)),
        (ValueError, lambda: seqs.next_tokens(ids[:3])),
        (IndexError, lambda: PackedSequences(offsets([0, 3, 2], device), 3).positions.cpu()),
        (IndexError, lambda: PackedSequences(offsets([0, 4], device), 3).positions.cpu()),
        (IndexError, lambda: PackedSequences(offsets([-1, 3], device), 3).positions.cpu()),
    ):
        with pytest.raises(kind):
            call()


def test_attention_refusals(device):
    at, x = cases.inputs([5, 4], 4, 2, 16, F32)
    q, k, v, _ = (y.to(device) for y in x)
    seqs = PackedSequences(offsets(at, device), 9)
    att = ops.packed_attention
    for kind, call in (
        (TypeError, lambda: att(q, k, v, offsets(at, device))),
        (ValueError, lambda: att(q, k, v, PackedSequences(offsets(at, device), 10))),
        (ValueError, lambda: att(q[:, :3], k, v, seqs)),
        (ValueError, lambda: att(q, k, v[:, :, :8], seqs)),
        (ValueError, lambda: att(q[None], k[None], v[None], seqs)),
        (ValueError, lambda: att(q[:, :, :8], k, v, seqs)),
        (ValueError, lambda: att(q[:8], k[:8], v[:8], seqs)),
        (ValueError, lambda: att(q, k[:, :0], v[:, :0], seqs)),
        (TypeError, lambda: att(q, k.bfloat16(), v.bfloat16(), seqs)),
        (ValueError, lambda: att(q, k, v, seqs, window=-1)),
        (ValueError, lambda: att(q, k, v, seqs, scale=float("nan"))),
        (ValueError, lambda: att(q, k, v, seqs, scale=float("inf"))),
        (ValueError, lambda: att(q, k, v, seqs, scale=1e39)),
    ):
        with pytest.raises(kind):
            call()
    if device == "mojo":
        with pytest.raises(ValueError):
            att(q, k, v, PackedSequences(offsets(at, "cpu"), 9))
        for bad in (q.double(), q[:, :, :12]):
            with pytest.raises(NotImplementedError):
                att(bad, bad, bad, seqs)


def test_a_gradient_of_the_gradient_is_refused(mojo):
    if mojo != "host":
        pytest.skip("the stand-in is for machines without a GPU")
    at, x = cases.inputs([5], 2, 2, 16, F32)
    q, k, v = (y.to("mojo").requires_grad_() for y in x[:3])
    dq, = torch.autograd.grad(ops.packed_attention(q, k, v, PackedSequences(offsets(at, "mojo"), 5)).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="second time"):
        dq.sum().backward()


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
def test_frequencies():
    plain = rotary_frequencies(8, 100.0, device="cpu")
    assert plain.scale == 1.0
    assert torch.allclose(plain.frequencies, torch.tensor([1, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15)
    linear = rotary_frequencies(8, 100.0, scaling="linear", factor=4.0, device="cpu").frequencies
    assert torch.equal(linear * 4, plain.frequencies)
    larger = rotary_frequencies(8, 100.0, scaling="base", factor=4.0, device="cpu").frequencies
    assert larger[0] == 1 and math.isclose(larger[-1] * 4, plain.frequencies[-1], rel_tol=1e-12)
    # 8 channels over 4096 positions: 652, 206, 65 and 21 turns; the ends of the mix
    # are pairs floor and ceil of 8 ln(4096 / (turns 2 pi)) / (2 ln 100) for 32 and 1
    parts = rotary_frequencies(8, 100.0, scaling="parts", factor=4.0, length=4096, device="cpu")
    low, high = math.floor(4 * math.log(4096 / (64 * math.pi)) / math.log(100)), math.ceil(4 * math.log(4096 / (2 * math.pi)) / math.log(100))
    mix = [min(max((j - low) / (high - low), 0), 1) for j in range(4)]
    want = [f * (1 - m) + f / 4 * m for f, m in zip(plain.frequencies.tolist(), mix)]
    assert torch.allclose(parts.frequencies, torch.tensor(want, dtype=torch.float64), rtol=1e-14)
    assert math.isclose(parts.scale, 1 + 0.1 * math.log(4))
    for kw in (dict(turned=7), dict(turned=0), dict(base=1.0), dict(factor=0.5), dict(scaling="unknown"), dict(scaling="parts"),
               dict(scaling="base", turned=2), dict(scaling="parts", length=100, slow=3, fast=2)):
        with pytest.raises(ValueError):
            rotary_frequencies(**{"turned": 8, "device": "cpu", **kw})


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n", [16, 6])
def test_rotary(device, interleaved, n):
    f = rotary_frequencies(n, device="cpu").frequencies
    g = torch.Generator().manual_seed(0)
    x = [torch.randn(2, 5, h, 16, generator=g).transpose(1, 2) for h in (3, 1, 3, 1)]
    for pos in (torch.arange(5) + 1000000, torch.randint(0, 99, (2, 5), generator=g, dtype=torch.int32)):
        q, k = (y.detach().to(device).requires_grad_() for y in x[:2])
        got = ops.rotary_at(q, k, pos.to(device), f.to(device), interleaved=interleaved, scale=1.5)
        torch.autograd.backward(got, [y.to(device) for y in x[2:]])
        for y, z, inverse in ((got[0], x[0], False), (got[1], x[1], False), (q.grad, x[2], True), (k.grad, x[3], True)):
            check(y, *logprob_cases.turned(z, pos, f, interleaved, 1.5, inverse))
    one = x[0][0].transpose(0, 1)
    got = ops.rotary_at(None, one.to(device), torch.arange(5).to(device), f.to(device), interleaved=interleaved)
    assert got[0] is None
    check(got[1].transpose(0, 1)[None], *logprob_cases.turned(x[0][:1], torch.arange(5), f, interleaved, 1.0))


def test_rotary_is_the_tables_rotation(device):
    """rotary_embedding's half layout, with the tables of the same angles."""
    f = rotary_frequencies(16, device="cpu").frequencies
    x = torch.randn(1, 2, 9, 16, generator=torch.Generator().manual_seed(1))
    angle = torch.arange(9)[:, None] * f
    cos, sin = (torch.cat([y, y], -1).float() for y in (angle.cos(), angle.sin()))
    want = ops.rotary_embedding(x, cos, sin)
    got = ops.rotary_at(x.to(device), None, torch.arange(9).to(device), f.to(device))[0]
    check(got, want.double().numpy(), np.full(x.shape, 2e-6))  # two roundings of the angles' sines and products, |x| < 5


def test_rotary_refusals(device):
    f = rotary_frequencies(16, device="cpu").frequencies.to(device)
    q, k = torch.zeros(2, 4, 5, 16).to(device), torch.zeros(2, 1, 5, 16).to(device)
    pos = torch.arange(5).to(device)
    at = ops.rotary_at
    for kind, call in (
        (ValueError, lambda: at(None, None, pos, f)),
        (ValueError, lambda: at(q[0, 0], None, pos, f)),
        (ValueError, lambda: at(q, k[:1], pos, f)),
        (ValueError, lambda: at(q, k[:, :, :4], pos, f)),
        (ValueError, lambda: at(q, k[..., :8], pos, f[:4])),
        (TypeError, lambda: at(q, k.bfloat16(), pos, f)),
        (ValueError, lambda: at(q, k, pos[:4], f)),
        (ValueError, lambda: at(q, k, pos.float(), f)),
        (ValueError, lambda: at(q, k, pos[None], f)),
        (ValueError, lambda: at(q, k, pos, f.float())),
        (ValueError, lambda: at(q[..., :14], None, pos, f)),
        (ValueError, lambda: at(q, k, pos, f[None])),
        (ValueError, lambda: at(q, k, pos, f, scale=float("inf"))),
    ):
        with pytest.raises(kind):
            call()
    if device == "mojo":
        with pytest.raises(NotImplementedError):
            at(q.double(), None, pos, f)
        with pytest.raises(ValueError):
            at(q, k, pos.cpu(), f)


# ---------------------------------------------------------------------------
# token log-probabilities
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("n,c,top", [(3, 7, 7), (5, 40, 3), (1, 1, 1), (4, 33, 0)])
def test_logprobs(device, n, c, top):
    x, tokens = logprob_cases.logits(n, c, F32)
    g = torch.Generator().manual_seed(3)
    grads = [torch.randn(n, generator=g), torch.randn(n, generator=g), torch.randn(n, top, generator=g) if top else None]
    if n > 2:
        tokens[1] = -100
    want = logprob_cases.expected(x, tokens, top, grads)
    leaf = x.to(device).requires_grad_()
    got = ops.token_logprobs(leaf, tokens.to(device), top=top, entropy=True)
    ends = [(y, z) for y, z in zip(got[:3], grads) if z is not None]
    torch.autograd.backward([y for y, _ in ends], [z.to(device) for _, z in ends])
    for name, y in (("logprobs", got.logprobs), ("entropy", got.entropy), ("top_logprobs", got.top_logprobs), ("dx", leaf.grad)):
        if y is not None:
            check(y, *want[name], name)
    if top:
        assert np.array_equal(got.top_tokens.cpu().numpy(), want["top_tokens"])
    assert ops.token_logprobs(x.to(device)).logprobs is None


def test_logprobs_of_shapes(device):
    x, tokens = logprob_cases.logits(6, 11, F32)
    got = ops.token_logprobs(x.view(2, 3, 11).to(device), tokens.view(2, 3).to(device), top=2, entropy=True)
    assert [tuple(y.shape) for y in got] == [(2, 3), (2, 3), (2, 3, 2), (2, 3, 2)]
    assert ops.token_logprobs(x[:0].to(device), tokens[:0].to(device), top=2).top_tokens.shape == (0, 2)


def test_logprobs_refusals(device):
    x, tokens = (y.to(device) for y in logprob_cases.logits(4, 11, F32))
    lp = ops.token_logprobs
    for kind, call in (
        (ValueError, lambda: lp(x, tokens[:3])),
        (ValueError, lambda: lp(x, tokens.int())),
        (ValueError, lambda: lp(x, tokens, top=12)),
        (ValueError, lambda: lp(x, tokens, top=-1)),
        (ValueError, lambda: lp(x[:, :0], tokens)),
        (ValueError, lambda: lp(x[0, 0])),
        (TypeError, lambda: lp(x.long(), tokens)),
        (IndexError, lambda: lp(x, tokens * 0 + 11).logprobs.cpu()),
        (IndexError, lambda: lp(x, tokens * 0 - 1).logprobs.cpu()),
    ):
        with pytest.raises(kind):
            call()
    if device == "mojo":
        with pytest.raises(NotImplementedError):
            lp(torch.zeros(2, 99).to("mojo"), top=65)
        with pytest.raises(NotImplementedError):
            lp(x.double())
        with pytest.raises(ValueError):
            lp(x, tokens.cpu())


# ---------------------------------------------------------------------------
# the models
# ---------------------------------------------------------------------------
LENGTHS = [9, 1, 0, 17, 4]


def packed(rows=33, device="cpu"):
    idx = torch.randint(0, 97, (rows,), generator=torch.Generator().manual_seed(2))
    return idx.to(device), PackedSequences.of_lengths(LENGTHS, rows, device=device)


def test_gemma_of_packed_sequences(device):
    """Each sequence's logits and gradients are those of a batch of it alone."""
    m, ref = decode_cases.model(F32, device, sinks=0)
    idx, seqs = packed(device=device)
    got = m.forward_packed(idx, seqs)
    at = [0, *itertools.accumulate(LENGTHS)]
    loss = 0.0
    for a, b in itertools.pairwise(at):
        if a < b:
            alone = ref(idx[a:b].cpu()[None])[0]
            check(got[a:b], alone.detach().numpy(), np.full(alone.shape, 1e-5 * alone.abs().max().item()))
            loss = loss + ops.token_logprobs(alone[:-1], idx[a + 1:b].cpu()).logprobs.sum()
    loss.backward()
    m.score_packed(idx, seqs).logprobs.sum().backward()
    for (name, p), r in zip(m.named_parameters(), ref.parameters()):
        check(p.grad, r.grad.numpy(), np.full(r.shape, 2e-5 * max(1.0, r.grad.abs().max().item())), name)


def test_gemma_scores(device):
    m, ref = decode_cases.model(F32, device, sinks=0)
    idx, seqs = packed(device=device)
    with torch.no_grad():
        got = m.score_packed(idx, seqs, top=3, entropy=True)
        want = ops.token_logprobs(ref.forward_packed(*packed()), packed()[1].next_tokens(packed()[0]), top=3, entropy=True)
    for y, z in zip(got[:3], want[:3]):
        check(y, z.numpy(), np.full(z.shape, 1e-4))
    assert torch.equal(got.top_tokens.cpu(), want.top_tokens)
    sinks, _ = decode_cases.model(F32, device, sinks=2)
    with pytest.raises(NotImplementedError, match="sinks"):
        sinks.forward_packed(idx, seqs)


def test_stretched_global_layers(device):
    """The factor goes through all three forwards alike."""
    cfg = Gemma3Config(vocab_size=97, hidden=32, layers=2, heads=2, kv_heads=1, head_dim=16, d_ff=32, window=4, global_every=2,
                       rope_global_factor=8.0)
    torch.manual_seed(0)
    m = Gemma3(cfg).to(device)
    idx = torch.randint(0, 97, (12,), generator=torch.Generator().manual_seed(2)).to(device)
    with torch.no_grad():
        a = m(idx[None])[0]
        b = m.forward_packed(idx, PackedSequences.of_lengths([12], device=device))
        plain = Gemma3(Gemma3Config(**{**cfg.__dict__, "rope_global_factor": 1.0})).to(device)
        plain.load_state_dict(m.state_dict())
        c = plain(idx[None])[0]
    assert (a - b).abs().max().item() < 1e-4 and (a - c).abs().max().item() > 1e-4


def gpt(device):
    torch.manual_seed(0)
    return GPT(GPTConfig(block_size=20, vocab_size=97, n_layer=2, n_head=2, n_embd=32)).to(device)


def test_gpt_of_packed_documents(device):
    m, ref = gpt(device), gpt("cpu").double()
    idx, seqs = packed(device=device)
    logits, loss = m(idx, seqs.next_tokens(idx, -1), seqs)
    loss.backward()
    at, total, rows = [0, *itertools.accumulate(LENGTHS)], 0.0, 0
    for a, b in itertools.pairwise(at):
        if b > a:
            alone, _ = ref(idx[a:b].cpu()[None])
            check(logits[a:b], alone[0].detach().numpy(), np.full(alone[0].shape, 1e-5))
        if b > a + 1:
            total = total + torch.nn.functional.cross_entropy(alone[0, :-1], idx[a + 1:b].cpu(), reduction="sum")
            rows += b - a - 1
    (total / rows).backward()
    assert abs(loss.item() - (total / rows).item()) < 1e-5
    for (name, p), r in zip(m.named_parameters(), ref.parameters()):
        check(p.grad, r.grad.numpy(), np.full(r.shape, 2e-6 + 2e-5 * r.grad.abs().max().item()), name)


def test_a_training_step_of_documents(device):
    m = gpt(device)
    idx, seqs = packed(device=device)
    opt = m.configure_optimizers(0.1, 1e-2, (0.9, 0.95), fused=device == "mojo")
    before = [p.detach().cpu().clone() for p in m.parameters()]
    loss = training_step(m, opt, idx, seqs.next_tokens(idx, -1), device_type=device, sequences=seqs)
    assert math.isfinite(loss.item())
    assert any(not torch.equal(p.detach().cpu(), b) for p, b in zip(m.parameters(), before))
