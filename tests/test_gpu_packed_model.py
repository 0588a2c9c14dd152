"""Packed sequences through the models on the MI355X, and the operators one
after another in a captured graph."""

import itertools
import math

import pytest
import torch

import decode_cases
from abi import CODE, call, i64, lib, p
from torch_mojo_backend import ops
from torch_mojo_backend.gpt2 import GPT, GPTConfig, training_step
from torch_mojo_backend.packing import PackedSequences

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _mojo(mojo):
    return mojo


LENGTHS = [90, 1, 0, 133, 64, 30]


def packed(rows=330, device="mojo"):
    idx = torch.randint(0, 97, (rows,), generator=torch.Generator().manual_seed(2))
    return idx.to(device), PackedSequences.of_lengths(LENGTHS, rows, device=device)


def close(got, want, lim, what):
    off = (got.detach().cpu().double() - want.detach().double()).abs().max()
    assert off <= lim * want.abs().max(), (what, off.item(), want.abs().max().item())


@pytest.mark.parametrize("dtype,head_dim,window", [(F32, 64, 7), (BF, 64, 40), (BF, 256, 100), (BF, 96, 64)])
def test_gemma(dtype, head_dim, window):
    """Logits and gradients of each parameter against the f64 model's.  A layer
    has six roundings of its rows between the residual sums and about as many in
    the backward: three layers and the head, 24 half steps of each in the norm, and
    in single entries four times that."""
    m, ref = decode_cases.model(dtype, "mojo", head_dim=head_dim, window=window, sinks=0)
    u = {F32: 2.0 ** -24, BF: 2.0 ** -8}[dtype]
    lim = 24 * u if dtype is BF else 24 * 16 * u  # (f32: sums of up to 256 products)
    idx, seqs = packed()
    cpu = packed(device="cpu")
    got, want = m.forward_packed(idx, seqs), ref.forward_packed(*cpu)
    close(got, want, lim, "logits")
    ops.token_logprobs(got, seqs.next_tokens(idx)).logprobs.sum().backward()
    ops.token_logprobs(want, cpu[1].next_tokens(cpu[0])).logprobs.sum().backward()
    for (name, x), r in zip(m.named_parameters(), ref.parameters()):
        off = (x.grad.cpu().double() - r.grad).norm() / r.grad.norm()
        assert off <= 4 * lim, (name, off.item())


def test_gemma_scores():
    m, ref = decode_cases.model(F32, "mojo", sinks=0)
    idx, seqs = packed()
    with torch.no_grad():
        got = m.score_packed(idx, seqs, top=4, entropy=True)
        cpu = packed(device="cpu")
        want = ref.score_packed(*cpu, top=4, entropy=True)
    for y, z, name in zip(got[:3], want[:3], got._fields):
        close(y, z, 1e-4, name)
    assert (got.top_tokens.cpu() == want.top_tokens).float().mean() > 0.99  # f32 may order a near tie either way


def test_of_no_rows_and_of_other_batches():
    """One model, batches one after another, one of no rows among them."""
    m, ref = decode_cases.model(F32, "mojo", sinks=0)
    for lengths, rows in (([5, 0, 9], 14), ([], 0), ([], 3), ([64, 1], 70)):
        idx = torch.randint(0, 97, (rows,), generator=torch.Generator().manual_seed(rows))
        with torch.no_grad():
            got = m.score_packed(idx.to("mojo"), PackedSequences.of_lengths(lengths, rows), top=1, entropy=True)
            want = ref.score_packed(idx, PackedSequences.of_lengths(lengths, rows, device="cpu"), top=1, entropy=True)
        assert got.logprobs.shape == (rows,) and got.top_tokens.shape == (rows, 1)
        if rows:
            close(got.logprobs, want.logprobs, 1e-4, "logprobs") if lengths else None
            close(got.entropy, want.entropy, 1e-4, "entropy")


@pytest.mark.parametrize("autocast", [None, BF])
def test_gpt_training_steps(autocast):
    """Documents packed end to end: loss and gradients are those of the f64 model,
    and a few steps run."""
    torch.manual_seed(0)
    cfg = GPTConfig(block_size=140, vocab_size=97, n_layer=2, n_head=2, n_embd=128)
    m, ref = GPT(cfg).to("mojo"), GPT(cfg).double()
    ref.load_state_dict({n: x.detach().cpu().double() for n, x in m.state_dict().items()})
    idx, seqs = packed()
    cpu = packed(device="cpu")
    _, want = ref(cpu[0], cpu[1].next_tokens(cpu[0], -1), cpu[1])
    want.backward()
    with torch.autocast("mojo", dtype=BF, enabled=autocast is not None):
        _, loss = m(idx, seqs.next_tokens(idx, -1), seqs)
    loss.backward()
    lim = 24 * 2.0 ** -8 if autocast else 1e-4  # (half steps of bf16 as above; f32 sums)
    assert abs(loss.item() - want.item()) <= lim * want.item()
    for (name, x), r in zip(m.named_parameters(), ref.parameters()):
        off = (x.grad.cpu().double() - r.grad).norm() / r.grad.norm()
        assert off <= 4 * lim, (name, off.item())
    opt = m.configure_optimizers(0.1, 1e-3, (0.9, 0.95))
    opt.zero_grad(set_to_none=True)
    for _ in range(3):
        loss = training_step(m, opt, idx, seqs.next_tokens(idx, -1), autocast, sequences=seqs)
        assert math.isfinite(loss.item())


def test_captured_with_other_sequences():
    """Plan, rotation, attention, scores and their backward as one graph, on a
    stream of its own: each replay takes the offsets, rows and logits of its time,
    and gives what the calls give by themselves."""
    t, h, hk, d, n, c, top = 500, 4, 2, 64, 6, 1000, 3
    g = torch.Generator().manual_seed(5)
    dev = "cuda"
    L = lib()

    def buffers():
        z = lambda *s, dt=BF: torch.zeros(*s, dtype=dt, device=dev)  # noqa: E731
        return dict(plan=z(L.mi355x_packed_plan_bytes(n, t), dt=torch.uint8), pos=z(t, dt=torch.int32), error=z(1, dt=torch.int32),
                    q1=z(t, h, d), k1=z(t, hk, d), out=z(t, h, d), low=z(t, h, d), lse=z(h, t, dt=F32), dq=z(t, h, d), dk=z(t, hk, d),
                    dv=z(t, hk, d), dq1=z(t, h, d), dk1=z(t, hk, d),
                    ws=z(L.mi355x_packed_attn_bwd_workspace_bytes(n, t, h, hk, d), dt=torch.uint8), lp=z(t, dt=F32), ent=z(t, dt=F32),
                    stats=z(t, 2, dt=F32), tlp=z(t, top, dt=F32), tt=z(t, top, dt=torch.int64), dx=z(t, 1000),
                    lws=z(max(L.mi355x_token_logprobs_workspace_bytes(t, c, top, 1), 16), dt=torch.uint8))

    x = dict(q=torch.zeros(t, h, d), k=torch.zeros(t, hk, d), v=torch.zeros(t, hk, d), dy=torch.zeros(t, h, d), logits=torch.zeros(t, c))
    x = {name: y.to(BF).to(dev) for name, y in x.items()}
    offsets, tokens = torch.zeros(n + 1, dtype=torch.int32, device=dev), torch.zeros(t, dtype=torch.int64, device=dev)
    freq = (10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)).to(dev)
    glp, gent = torch.randn(t, generator=g).to(dev), torch.randn(t, generator=g).to(dev)

    def run(b, stream):
        th = lambda y: i64(*y.stride()[:2])  # noqa: E731
        bht = lambda y: i64(0, y.stride(1), y.stride(0))  # noqa: E731
        call("mi355x_packed_plan", p(b["plan"]), b["plan"].numel(), p(b["pos"]), p(offsets), n, t, p(b["error"]), stream)
        call("mi355x_rope_at", p(b["q1"]), bht(b["q1"]), p(x["q"]), bht(x["q"]), h, p(b["k1"]), bht(b["k1"]), p(x["k"]), bht(x["k"]), hk,
             p(b["pos"]), CODE[torch.int32], 0, p(freq), 1, t, d, d, 0, 1.0, 0, CODE[BF], stream)
        call("mi355x_packed_attn_fwd", p(b["out"]), th(b["out"]), p(b["low"]), p(b["lse"]), p(b["q1"]), th(b["q1"]), p(b["k1"]), th(b["k1"]),
             p(x["v"]), th(x["v"]), p(b["plan"]), n, t, h, hk, d, 0.125, 0, CODE[BF], stream)
        call("mi355x_packed_attn_bwd", p(b["dq"]), th(b["dq"]), p(b["dk"]), th(b["dk"]), p(b["dv"]), th(b["dv"]), p(x["dy"]), th(x["dy"]),
             p(b["q1"]), th(b["q1"]), p(b["k1"]), th(b["k1"]), p(x["v"]), th(x["v"]), p(b["out"]), th(b["out"]), p(b["low"]), p(b["lse"]),
             p(b["plan"]), n, t, h, hk, d, 0.125, 0, CODE[BF], p(b["ws"]), b["ws"].numel(), stream)
        call("mi355x_rope_at", p(b["dq1"]), bht(b["dq1"]), p(b["dq"]), bht(b["dq"]), h, p(b["dk1"]), bht(b["dk1"]), p(b["dk"]), bht(b["dk"]),
             hk, p(b["pos"]), CODE[torch.int32], 0, p(freq), 1, t, d, d, 0, 1.0, 1, CODE[BF], stream)
        call("mi355x_token_logprobs_fwd", p(b["lp"]), p(b["ent"]), p(b["stats"]), p(b["tlp"]), p(b["tt"]), p(x["logits"]), CODE[BF], c,
             p(tokens), t, c, top, -100, p(b["error"]), p(b["lws"]), b["lws"].numel(), stream)
        call("mi355x_token_logprobs_bwd", p(b["dx"]), 1000, p(x["logits"]), CODE[BF], c, p(b["stats"]), p(b["ent"]), p(tokens), p(b["tt"]),
             top, p(glp), p(gent), None, t, c, -100, stream)

    def fill(lengths):
        at = [0, *itertools.accumulate(lengths)]
        offsets.copy_(torch.tensor(at, dtype=torch.int32))
        tokens.copy_(torch.randint(0, c, (t,), generator=g))
        for y in x.values():
            y.copy_(torch.randn(*y.shape, generator=g).to(BF))

    captured, plain = buffers(), buffers()
    fill([100, 0, 50, 200, 1, 99])
    run(captured, None)  # (kernels are loaded before the capture)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        run(captured, side.cuda_stream)
    for lengths in ([100, 0, 50, 200, 1, 99], [500, 0, 0, 0, 0, 0], [1, 1, 1, 1, 1, 1], [0, 0, 0, 0, 0, 0], [64, 128, 63, 129, 65, 51]):
        fill(lengths)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        run(plain, None)
        torch.cuda.synchronize()
        assert not captured["error"].item()
        # (a plan's order within a tile number is free, and workspaces hold what a call leaves)
        for name in plain.keys() - {"plan", "ws", "lws"}:
            live = slice(None) if name not in ("low",) else slice(0, sum(lengths))
            assert torch.equal(captured[name][live], plain[name][live]), (name, lengths)
