"""What the operators of packed sequences are measured on: turning queries and
keys by the angles of their positions, causal attention over sequences of
different lengths laid end to end, and log-probabilities of given tokens with
entropy and top alternatives; forward, and backward where a program trains.

A case is a dict of plain values; `kind` names the operator.  Sequence i of a
packed batch is rows offsets[i] .. offsets[i + 1] - 1; rows behind the last one
are padding, whose results are zero.  Where `own` is false, `run` is the plain
form in elementary torch operations.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False


def listed():
    return [
        # the queries and keys of one new token in a Gemma-3-1B-shaped layer:
        # the smallest call of a decode step, where latency counts
        {"name": "rotary_token_bf16", "kind": "rotary", "dtype": "bf16", "batch": 1, "tokens": 1, "heads": 4,
         "kv_heads": 1, "head_dim": 256, "turned": 256, "interleaved": False, "start": 8000, "factor": 1.0,
         "train": False},
        # a padded batch far into a stretched context: part of the head,
        # neighbouring channels paired, f32, an odd length
        {"name": "rotary_far_f32", "kind": "rotary", "dtype": "f32", "batch": 2, "tokens": 1021, "heads": 12,
         "kv_heads": 12, "head_dim": 64, "turned": 32, "interleaved": True, "start": 1000003, "factor": 16.0,
         "train": False},
        # grouped heads of a training batch, forward and backward
        {"name": "rotary_train_bf16", "kind": "rotary", "dtype": "bf16", "batch": 4, "tokens": 4096, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "turned": 128, "interleaved": False, "start": 0, "factor": 8.0,
         "train": True},
        # a few short prompts through GPT-2 small's heads at once, where
        # latency counts
        {"name": "packed_prompts_bf16", "kind": "attention", "dtype": "bf16", "tokens": 333, "sequences": 8,
         "spread": 2.0, "tail": 0, "heads": 12, "kv_heads": 12, "head_dim": 64, "window": 0, "train": False},
        # longer prompts of a head_dim between the powers of two, f16
        {"name": "packed_prompts_f16", "kind": "attention", "dtype": "f16", "tokens": 6001, "sequences": 5,
         "spread": 1.5, "tail": 0, "heads": 16, "kv_heads": 4, "head_dim": 96, "window": 0, "train": False},
        # a small f32 training batch of GPT-2 small's heads, odd lengths, a
        # tail of padding
        {"name": "packed_train_f32", "kind": "attention", "dtype": "f32", "tokens": 1021, "sequences": 6,
         "spread": 1.5, "tail": 37, "heads": 12, "kv_heads": 12, "head_dim": 64, "window": 0, "train": True},
        # GPT-2 small's heads trained on a batch of 16 x 1024 tokens of
        # documents, most of them short
        {"name": "packed_train_documents", "kind": "attention", "dtype": "bf16", "tokens": 16384, "sequences": 48,
         "spread": 3.0, "tail": 100, "heads": 12, "kv_heads": 12, "head_dim": 64, "window": 0, "train": True},
        # a Gemma-3-1B-shaped local layer fine-tuned on three sequences
        {"name": "packed_train_gemma", "kind": "attention", "dtype": "bf16", "tokens": 4096, "sequences": 3,
         "spread": 1.0, "tail": 0, "heads": 4, "kv_heads": 1, "head_dim": 256, "window": 512, "train": True},
        # grouped heads trained on a few long sequences
        {"name": "packed_train_long", "kind": "attention", "dtype": "bf16", "tokens": 16384, "sequences": 4,
         "spread": 1.2, "tail": 0, "heads": 32, "kv_heads": 8, "head_dim": 128, "window": 0, "train": True},
        # the token that a Gemma-3-shaped model answers with, and what else it
        # might have been
        {"name": "logprobs_token_bf16", "kind": "logprobs", "dtype": "bf16", "tokens": 1, "vocab": 262144, "top": 20,
         "entropy": False, "train": False},
        # scoring of 1000 positions from f32 logits of GPT-2's vocabulary
        {"name": "logprobs_score_f32", "kind": "logprobs", "dtype": "f32", "tokens": 1000, "vocab": 50257, "top": 5,
         "entropy": True, "train": False},
        # 8 x 1024 positions of a policy's training step with an entropy term
        {"name": "logprobs_train_bf16", "kind": "logprobs", "dtype": "bf16", "tokens": 8192, "vocab": 50257, "top": 0,
         "entropy": True, "train": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _largest(kind):
    return max(work(c)["flops"] for c in listed() if c["kind"] == kind)


def draw(rng):
    kind = rng.choice(["rotary", "attention", "attention", "attention", "logprobs", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "logprobs":
        vocab = _log_int(rng, 1000, 262144)
        tokens = _log_int(rng, 1, max(1, min(8192, 8192 * 50257 // (vocab * (2 if dtype == "f32" else 1)))))
        train = rng.random() < 0.5
        return {"kind": kind, "dtype": dtype, "tokens": tokens, "vocab": vocab,
                "top": rng.choice([0, 0, 1]) if train else rng.choice([0, 1, 5, 5, 20, 32]),
                "entropy": rng.random() < 0.6, "train": train}
    head_dim = rng.choice([64, 64, 80, 96, 128, 128, 256])
    kv_heads, group = rng.choice([1, 2, 4, 8, 12]), rng.choice([1, 1, 2, 4, 8])
    if kind == "rotary":
        tokens = _log_int(rng, 1, 8192)
        heads = kv_heads * group
        most = 4 * 4096 * 40 * 128 // (2 if dtype == "f32" else 1)
        batch = _log_int(rng, 1, max(1, min(32, most // (tokens * (heads + kv_heads) * head_dim))))
        tokens = max(1, min(tokens, most // (batch * (heads + kv_heads) * head_dim)))
        return {"kind": kind, "dtype": dtype, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
                "head_dim": head_dim, "turned": head_dim // rng.choice([1, 1, 1, 2]),
                "interleaved": rng.random() < 0.4, "start": rng.choice([0, 0, _log_int(rng, 1, 4000000)]),
                "factor": rng.choice([1.0, 1.0, 4.0, 8.0, 32.0]), "train": rng.random() < 0.6}
    tokens = _log_int(rng, 1, 16384)
    c = {"kind": kind, "dtype": dtype, "tokens": tokens, "sequences": _log_int(rng, 1, min(tokens, 200)),
         "spread": rng.choice([0.0, 1.0, 2.0, 4.0]), "tail": rng.choice([0, 0, 0, min(1, tokens - 1), tokens // 9]),
         "heads": kv_heads * group, "kv_heads": kv_heads, "head_dim": head_dim,
         "window": rng.choice([0, 0, 0, _log_int(rng, 1, 4096)]), "train": rng.random() < 0.6}
    most = _largest(kind) / (16 if dtype == "f32" else 1)
    while work(dict(c, window=0))["flops"] > most:  # the plain form computes what a window hides, too
        if c["heads"] > c["kv_heads"]:
            c["heads"] -= c["kv_heads"]
        elif c["heads"] > 1:
            c["heads"] = c["kv_heads"] = c["heads"] // 2
        else:
            c["sequences"] += 1
    return c


# ---------------------------------------------------------------------------
# lengths, from the case alone, and inputs, from the seed
# ---------------------------------------------------------------------------
def _dtype(case):
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[case["dtype"]]


def _offsets(case):
    """Where the sequences begin: lengths spread over a factor of e ** spread,
    the third of five and more empty, `tail` rows of padding behind the last."""
    n, rows = case["sequences"], max(0, case["tokens"] - case["tail"])
    share = [math.exp(-case["spread"] * ((i * 0.6180339887 + 0.1) % 1.0)) for i in range(n)]
    if n >= 5:
        share[2] = 0.0
    total, at, out = sum(share), 0.0, [0]
    for s in share:
        at += s
        out.append(min(rows, round(rows * at / total)))
    return out


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _frequencies(case):
    """Radians a position of the turned channels' pairs, f64; a stretched
    context divides those of the slow pairs by its factor and, between 1 and 32
    turns over 4096 positions, part by part; and the length of the turned part."""
    n = case["turned"]
    freq = 10000.0 ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
    if case["factor"] == 1.0:
        return freq.cuda(), 1.0
    turns = 4096 * freq / (2 * math.pi)
    keep = ((turns - 1) / 31).clamp(0, 1)
    return (freq * keep + freq / case["factor"] * (1 - keep)).cuda(), 0.1 * math.log(case["factor"]) + 1.0


def _inputs(case, seed):
    """Every tensor of the call, dense."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 2654435761 % (1 << 62))
    dt, t = _dtype(case), case["tokens"]
    s = {}
    if case["kind"] == "logprobs":
        # a broad spread, and a few tokens that stand out of it
        logits = _randn(gen, t, case["vocab"]) * 2.0
        peaks = torch.randint(0, case["vocab"], (t, 8), generator=gen, device="cuda")
        logits.scatter_add_(1, peaks, 6.0 + 2.0 * _randn(gen, t, 8))
        s["logits"] = logits.to(dt)
        pick = torch.randint(0, 8, (t, 1), generator=gen, device="cuda")
        s["tokens"] = peaks.gather(1, pick)[:, 0]
        if case["train"]:
            s["d_logprobs"] = _randn(gen, t) / t
            if case["entropy"]:
                s["d_entropy"] = -0.01 * torch.rand(t, generator=gen, device="cuda") / t
            if case["top"]:
                s["d_top"] = _randn(gen, t, case["top"]) / t
        return s
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    lead = (case["batch"], t) if case["kind"] == "rotary" else (t,)
    s["q"], s["k"] = _randn(gen, *lead, h, d).to(dt), _randn(gen, *lead, hk, d).to(dt)
    if case["kind"] == "rotary":
        starts = torch.randint(0, case["start"] + 1, (case["batch"], 1), generator=gen, device="cuda")
        s["positions"] = (starts + torch.arange(t, device="cuda")).int()
        if case["train"]:
            s["d_q"], s["d_k"] = _randn(gen, *lead, h, d).to(dt), _randn(gen, *lead, hk, d).to(dt)
        return s
    s["v"] = _randn(gen, *lead, hk, d).to(dt)
    s["offsets"] = torch.tensor(_offsets(case), dtype=torch.int32, device="cuda")
    if case["train"]:
        s["d_out"] = _randn(gen, *lead, h, d).to(dt)
    return s


# ---------------------------------------------------------------------------
# what a program has in hand, and the call
# ---------------------------------------------------------------------------
def _mojo(t):
    """A tensor of the framework's device with the given values."""
    from torch_mojo_backend import TorchMojoTensor

    raw = t.contiguous().reshape(-1).view(torch.uint8)
    strides = tuple(t.contiguous().stride())
    return TorchMojoTensor._make(raw, raw.data_ptr(), tuple(t.shape), strides, 0, t.dtype, 0)


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "rotary":
        s["frequencies"], s["scale"] = _frequencies(case)
    if own:
        pkg = str(Path(__file__).resolve().parents[1] / "torch-mojo-backend_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from torch_mojo_backend import register_mojo_devices

        register_mojo_devices()
        s = {n: _mojo(t) if isinstance(t, torch.Tensor) else t for n, t in s.items()}
        if case["kind"] == "attention":  # one plan of a batch serves all of a model's layers
            from torch_mojo_backend.packing import PackedSequences

            s["sequences"] = PackedSequences(s["offsets"], case["tokens"])
    if case["kind"] == "rotary":  # heads in front, as views of a projection's output
        for n in ("q", "k", "d_q", "d_k"):
            if n in s:
                s[n] = s[n].transpose(1, 2)
    if own and case["train"]:
        for n in ("q", "k", "v", "logits"):
            if n in s:
                s[n].requires_grad_()
    s["case"] = dict(case)
    return s


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"rotary": _own_rotary, "attention": _own_attention, "logprobs": _own_logprobs}[kind](s)
    return {"rotary": _rotary, "attention": _attention, "logprobs": _logprobs}[kind](s)


def _own_rotary(s):
    from torch_mojo_backend import ops

    c = s["case"]
    for n in ("q", "k"):
        s[n].grad = None
    q, k = ops.rotary_at(s["q"], s["k"], s["positions"], s["frequencies"], interleaved=c["interleaved"],
                         scale=s["scale"])
    if not c["train"]:
        return {"q": q, "k": k}
    torch.autograd.backward((q, k), (s["d_q"], s["d_k"]))
    return {"q": q.detach(), "k": k.detach(), "d_q": s["q"].grad, "d_k": s["k"].grad}


def _own_attention(s):
    from torch_mojo_backend import ops

    c = s["case"]
    for n in ("q", "k", "v"):
        s[n].grad = None
    out = ops.packed_attention(s["q"], s["k"], s["v"], s["sequences"], window=c["window"])
    if not c["train"]:
        return {"out": out}
    out.backward(s["d_out"])
    return {"out": out.detach(), "d_q": s["q"].grad, "d_k": s["k"].grad, "d_v": s["v"].grad}


def _own_logprobs(s):
    from torch_mojo_backend import ops

    c = s["case"]
    s["logits"].grad = None
    r = ops.token_logprobs(s["logits"], s["tokens"], top=c["top"], entropy=c["entropy"])
    out = {"logprobs": r.logprobs.detach()}
    if c["entropy"]:
        out["entropy"] = r.entropy.detach()
    if c["top"]:
        out["top_logprobs"], out["top_tokens"] = r.top_logprobs.detach(), r.top_tokens
    if c["train"]:
        ends = [(r.logprobs, "d_logprobs"), (r.entropy, "d_entropy"), (r.top_logprobs, "d_top")]
        ends = [(x, s[n]) for x, n in ends if n in s]
        torch.autograd.backward([x for x, _ in ends], [g for _, g in ends])
        out["d_logits"] = s["logits"].grad
    return out


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------
def _turn(x, cos, sin, turned, interleaved):
    """x [batch, heads, tokens, d] with its first channels turned in pairs."""
    a, rest = x[..., :turned], x[..., turned:]
    if interleaved:
        even, odd = a[..., 0::2], a[..., 1::2]
        a = torch.stack([even * cos - odd * sin, odd * cos + even * sin], dim=-1).flatten(-2)
    else:
        low, high = a[..., :turned // 2], a[..., turned // 2:]
        a = torch.cat([low * cos - high * sin, high * cos + low * sin], dim=-1)
    return torch.cat([a, rest], dim=-1)


def _rotary(s):
    c = s["case"]
    angle = s["positions"][:, None, :, None].double() * s["frequencies"]
    cos, sin = (angle.cos() * s["scale"]).float(), (angle.sin() * s["scale"]).float()
    out = {n: _turn(s[n].float(), cos, sin, c["turned"], c["interleaved"]).to(s[n].dtype) for n in ("q", "k")}
    if c["train"]:
        for n in ("d_q", "d_k"):
            out[n] = _turn(s[n].float(), cos, -sin, c["turned"], c["interleaved"]).to(s[n].dtype)
    return out


def _attention(s):
    c = s["case"]
    q, k, v = s["q"], s["k"], s["v"]
    h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    scale = 1.0 / math.sqrt(d)
    out = {"out": torch.zeros_like(q)}
    if c["train"]:
        out.update(d_q=torch.zeros_like(q), d_k=torch.zeros_like(k), d_v=torch.zeros_like(v))
    at = _offsets(c)  # (the program laid the sequences out itself)
    for a, b in zip(at, at[1:]):
        if a == b:
            continue
        n = b - a
        i = torch.arange(n, device="cuda")
        hidden = i[None] > i[:, None]
        if c["window"]:
            hidden |= i[:, None] - i[None] >= c["window"]
        qs = q[a:b].float().view(n, hk, h // hk, d).permute(1, 2, 0, 3)
        ks, vs = (x[a:b].float().permute(1, 0, 2)[:, None] for x in (k, v))
        e = (qs @ ks.transpose(-1, -2)).mul_(scale).masked_fill_(hidden, -math.inf)
        e = e.sub_(e.amax(-1, keepdim=True)).exp_()
        p = e.div_(e.sum(-1, keepdim=True))
        o = p @ vs
        out["out"][a:b] = o.permute(2, 0, 1, 3).reshape(n, h, d).to(q.dtype)
        if c["train"]:
            do = s["d_out"][a:b].float().view(n, hk, h // hk, d).permute(1, 2, 0, 3)
            out["d_v"][a:b] = (p.transpose(-1, -2) @ do).sum(1).transpose(0, 1).to(q.dtype)
            ds = (do @ vs.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
            out["d_q"][a:b] = (ds @ ks).permute(2, 0, 1, 3).reshape(n, h, d).to(q.dtype)
            out["d_k"][a:b] = (ds.transpose(-1, -2) @ qs).sum(1).transpose(0, 1).to(q.dtype)
    return out


def _logprobs(s):
    c = s["case"]
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    logp = x - top
    logp -= torch.log(torch.exp(logp).sum(-1, keepdim=True))
    tokens = s["tokens"][:, None]
    out = {"logprobs": logp.gather(1, tokens)[:, 0]}
    p = torch.exp(logp) if c["entropy"] or c["train"] else None
    if c["entropy"]:
        out["entropy"] = -(p * logp).sum(-1)
    if c["top"]:
        order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :c["top"]]
        out["top_logprobs"], out["top_tokens"] = logp.gather(1, order), order
    if c["train"]:
        g = s["d_logprobs"][:, None]
        total = g + s["d_top"].sum(-1, keepdim=True) if c["top"] else g
        if c["entropy"]:
            d = (logp + out["entropy"][:, None]).mul_(s["d_entropy"][:, None]).add_(total).mul_(p).neg_()
        else:
            d = p.mul_(total).neg_()
        d.scatter_add_(1, tokens, g)
        if c["top"]:
            d.scatter_add_(1, out["top_tokens"], s["d_top"])
        out["d_logits"] = d.to(s["logits"].dtype)
    return out


# ---------------------------------------------------------------------------
# what one call cannot do without
# ---------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    t = case["tokens"]
    if case["kind"] == "logprobs":
        values = t * case["vocab"]
        small = t * (8 + 4 + 4 * case["entropy"] + 12 * case["top"])
        if case["train"]:  # logits in, their gradient out
            return {"bytes": 2 * values * e + small + 4 * t, "flops": 8.0 * values}
        return {"bytes": values * e + small, "flops": 4.0 * values}
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "rotary":
        rows = case["batch"] * t * (h + hk)
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 2 * rows * d * e + passes * 4 * case["batch"] * t,
                "flops": passes * 3.0 * rows * case["turned"]}
    at = _offsets(case)
    pairs = 0
    for a, b in zip(at, at[1:]):
        n = b - a
        w = min(n, case["window"]) if case["window"] else n
        pairs += w * (w + 1) // 2 + (n - w) * w
    rows = at[-1]
    if case["train"]:  # q, k, v, dO in; O, dQ, dK, dV out
        return {"bytes": 4 * (rows * h + rows * hk) * d * e, "flops": 14.0 * d * h * pairs}
    return {"bytes": 2 * (rows * h + rows * hk) * d * e, "flops": 4.0 * d * h * pairs}


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_rotary(case, s):
    freq, scale = _frequencies(case)
    n = case["turned"]
    j = torch.arange(n // 2, device="cuda")
    first, second = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + n // 2)
    angle = s["positions"].double()[..., None] * freq  # [batch, tokens, pairs]
    z = torch.polar(torch.full_like(angle, scale), angle)[:, :, None]

    def turn(x, z):
        y = x.double()
        w = torch.complex(y[..., first], y[..., second]) * z
        y = y.clone()
        y[..., first], y[..., second] = w.real, w.imag
        return y.transpose(1, 2)

    out = {"q": turn(s["q"], z), "k": turn(s["k"], z)}
    if case["train"]:
        out.update(d_q=turn(s["d_q"], z.conj()), d_k=turn(s["d_k"], z.conj()))
    return out


def _exact_attention(case, s):
    d, g, window = case["head_dim"], case["heads"] // case["kv_heads"], case["window"]
    got = {n: torch.zeros(s[x].shape, dtype=torch.float64, device="cuda")
           for n, x in (("out", "q"), ("d_q", "q"), ("d_k", "k"), ("d_v", "v"))}
    at = _offsets(case)
    for a, b in zip(at, at[1:]):
        if a == b:
            continue
        seen = torch.ones(b - a, b - a, dtype=torch.bool, device="cuda").tril()
        if window:
            seen = seen.triu(1 - window)
        for h in range(case["heads"]):
            q, k, v = (s[x][a:b, y].double().requires_grad_() for x, y in (("q", h), ("k", h // g), ("v", h // g)))
            w = torch.softmax(((q @ k.T) / math.sqrt(d)).masked_fill(~seen, -math.inf), dim=-1)
            out = w @ v
            got["out"][a:b, h] = out.detach()
            if case["train"]:
                dq, dk, dv = torch.autograd.grad(out, (q, k, v), s["d_out"][a:b, h].double())
                got["d_q"][a:b, h] = dq
                got["d_k"][a:b, h // g] += dk
                got["d_v"][a:b, h // g] += dv
    return got if case["train"] else {"out": got["out"]}


def _exact_logprobs(case, s):
    n, k = case["tokens"], case["top"]
    logprobs, entropy, tops, order, grads = [], [], [], [], []
    rows = max(1, (1 << 26) // case["vocab"])
    for a in range(0, n, rows):
        x = s["logits"][a:a + rows].double().requires_grad_(case["train"])
        logp = torch.log_softmax(x, dim=-1)
        picked = logp[torch.arange(x.shape[0], device="cuda"), s["tokens"][a:a + rows]]
        logprobs.append(picked.detach())
        ends = [(picked, "d_logprobs")]
        if case["entropy"]:
            h = -(torch.exp(logp) * logp).sum(-1)
            entropy.append(h.detach())
            ends.append((h, "d_entropy"))
        if k:
            order.append(torch.sort(x.detach(), dim=-1, descending=True, stable=True)[1][:, :k])
            best = logp.gather(1, order[-1])
            tops.append(best.detach())
            ends.append((best, "d_top"))
        if case["train"]:
            grads.append(torch.autograd.grad([y for y, _ in ends], x, [s[g][a:a + rows].double() for _, g in ends])[0])
    out = {"logprobs": torch.cat(logprobs)}
    if case["entropy"]:
        out["entropy"] = torch.cat(entropy)
    if k:
        out["top_logprobs"], out["top_tokens"] = torch.cat(tops), torch.cat(order)
    if case["train"]:
        out["d_logits"] = torch.cat(grads)
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    return {"rotary": _exact_rotary, "attention": _exact_attention, "logprobs": _exact_logprobs}[case["kind"]](case, s)
