"""What the serving and sliding-window operators are measured on: appending
rotated keys and values to a paged cache (16 or 32 bits, or 4 bits with a scale
and a minimum for each 32 channels), attention of new tokens over such a cache,
and attention over a sliding window with a few first tokens that stay visible
(sinks), forward and backward.

A case is a dict of plain values; `kind` names the operator.  Token t of
sequence b sits at position starts[b] + t; tokens from counts[b] on are
padding, and a sequence with no tokens is a place that no request fills.
Where `own` is false, `run` is the plain form in elementary torch operations.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

GROUP = 32  # channels that share a scale and a minimum in a 4-bit cache
LIMIT = 61440.0  # what it clamps to: every value it reads back is then finite in 16 bits


def listed():
    return [
        # one new token of one sequence in a Gemma-3-1B-shaped layer: the
        # smallest call of a decode step, where latency counts
        {"name": "append_token_bf16", "kind": "append", "dtype": "bf16", "bits": 16, "batch": 1, "tokens": 1,
         "heads": 4, "kv_heads": 1, "head_dim": 256, "page": 16, "context": 700, "rotate": True},
        # a padded batch of prompts of 12 x 64 heads (GPT-2 small's), learned
        # positions, so nothing is rotated; pages of 24 end inside any tile
        {"name": "append_prompts_f32", "kind": "append", "dtype": "f32", "bits": 16, "batch": 5, "tokens": 333,
         "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 24, "context": 333, "rotate": False},
        # four long prompts into a 4-bit cache, and their rows read back
        {"name": "append_prompts_4bit", "kind": "append", "dtype": "bf16", "bits": 4, "batch": 4, "tokens": 2048,
         "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64, "context": 2048, "rotate": True},
        # the decode step of one sequence in a Gemma-3-1B-shaped local layer
        # (window 512) with four sinks
        {"name": "decode_local_bf16", "kind": "decode", "dtype": "bf16", "bits": 16, "batch": 1, "tokens": 1,
         "heads": 4, "kv_heads": 1, "head_dim": 256, "page": 16, "context": 4096, "window": 512, "sinks": 4},
        # four drafted tokens verified for three sequences, f32, odd lengths
        {"name": "decode_drafts_f32", "kind": "decode", "dtype": "f32", "bits": 16, "batch": 3, "tokens": 4,
         "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 24, "context": 333, "window": 0, "sinks": 0},
        # a serving batch over long contexts, grouped heads
        {"name": "decode_batch_bf16", "kind": "decode", "dtype": "bf16", "bits": 16, "batch": 32, "tokens": 1,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "context": 16384, "window": 0, "sinks": 0},
        # the decode step of one sequence in a Gemma-3-1B-shaped global layer,
        # 4 bits, a length that divides nothing
        {"name": "decode_token_4bit", "kind": "decode", "dtype": "bf16", "bits": 4, "batch": 1, "tokens": 1,
         "heads": 4, "kv_heads": 1, "head_dim": 256, "page": 16, "context": 8191, "window": 0, "sinks": 0},
        # the serving batch again, over a 4-bit cache
        {"name": "decode_batch_4bit", "kind": "decode", "dtype": "bf16", "bits": 4, "batch": 32, "tokens": 1,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "context": 16384, "window": 0, "sinks": 0},
        # a short f32 training batch of GPT-2 small's heads, an odd length
        {"name": "window_train_f32", "kind": "window", "dtype": "f32", "batch": 2, "tokens": 255, "heads": 12,
         "kv_heads": 12, "head_dim": 64, "window": 64, "sinks": 1, "train": True},
        # a Gemma-3-1B-shaped local layer fine-tuned on a 4096-token sequence
        {"name": "window_train_gemma", "kind": "window", "dtype": "bf16", "batch": 1, "tokens": 4096, "heads": 4,
         "kv_heads": 1, "head_dim": 256, "window": 512, "sinks": 4, "train": True},
        # GPT-2 small's heads trained on a long sequence
        {"name": "window_train_long", "kind": "window", "dtype": "bf16", "batch": 1, "tokens": 8192, "heads": 12,
         "kv_heads": 12, "head_dim": 64, "window": 1024, "sinks": 4, "train": True},
        # two prompts through grouped heads without gradients
        {"name": "window_prefill_f16", "kind": "window", "dtype": "f16", "batch": 2, "tokens": 2000, "heads": 16,
         "kv_heads": 4, "head_dim": 128, "window": 512, "sinks": 8, "train": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "window"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    head_dim = rng.choice([64, 128, 128, 256])
    kv_heads, group = rng.choice([1, 2, 4, 8, 12]), rng.choice([1, 1, 2, 4, 8])
    if kind == "window":
        tokens = _log_int(rng, 1, 8192)
        # heads that fit into the largest listed case, over the whole batch
        most = max(1, 12 * 64 * 8192 * 8192 // (head_dim * tokens * tokens * (4 if dtype == "f32" else 1)))
        kv_heads = min(kv_heads, most)
        heads = kv_heads * min(group, most // kv_heads)
        return {"kind": kind, "dtype": dtype, "batch": _log_int(rng, 1, min(8, most // heads)), "tokens": tokens,
                "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "window": _log_int(rng, 16, 2048),
                "sinks": rng.choice([0, 1, 4, 4, 16, 70]), "train": rng.random() < 0.7}
    heads = kv_heads * group
    bits = rng.choice([16, 4])
    if bits == 4 and dtype == "f32":
        dtype = "bf16"
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    c = {"kind": kind, "dtype": dtype, "bits": bits, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
         "page": page}
    if kind == "append":
        tokens = _log_int(rng, 1, 2048)
        batch = _log_int(rng, 1, max(1, min(64, 4 * 2048 * 24 * 128 // (tokens * (heads + kv_heads) * head_dim))))
        return dict(c, batch=batch, tokens=tokens, context=tokens + rng.choice([0, 1, _log_int(rng, 1, 4096)]),
                    rotate=rng.random() < 0.75)
    tokens = rng.choice([1, 1, 1, 2, 4, 8])
    context = tokens + _log_int(rng, 1, 32768)
    most = 32 * 16384 * 8 * 128 // (2 if dtype == "f32" else 1)
    context = max(tokens, min(context, most // (kv_heads * head_dim)))
    batch = _log_int(rng, 1, max(1, min(64, most // (context * kv_heads * head_dim))))
    windowed = rng.random() < 0.4
    return dict(c, batch=batch, tokens=tokens, context=context, window=_log_int(rng, 16, 4096) if windowed else 0,
                sinks=rng.choice([0, 1, 4, 40]) if windowed else 0)


# ---------------------------------------------------------------------------
# lengths, from the case alone, and inputs, from the seed
# ---------------------------------------------------------------------------
def _dtype(case):
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[case["dtype"]]


def _lengths(case):
    """starts and counts of each sequence: contexts between half and the whole
    of case["context"], the last place of a batch of five and more empty."""
    starts, counts = [], []
    for i in range(case["batch"]):
        part = 1.0 - 0.5 * ((i * 0.6180339887) % 1.0)
        n = max(1, int(case["context"] * part))
        c = min(n, case["tokens"])
        starts.append(n - c)
        counts.append(c)
    if case["batch"] >= 5:
        starts[-1], counts[-1] = 0, 0
    return starts, counts


def _pages_each(case):
    return -(-case["context"] // case["page"])


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _packed(gen, shape):
    """Random codes and (scale, minimum) pairs of values about N(0, 1)."""
    *lead, d = shape
    codes = torch.randint(0, 256, (*lead, d // 2), generator=gen, device="cuda", dtype=torch.uint8)
    scale = (0.2 + 0.15 * torch.rand(*lead, d // GROUP, generator=gen, device="cuda")).half()
    low = (-7.5 * scale.float() + 0.2 * _randn(gen, *lead, d // GROUP)).half()
    return codes, torch.stack([scale, low], dim=-1)


def _tables(case):
    """cos, sin [positions, head_dim] of the rotation, f32 from 64-bit angles."""
    d, n = case["head_dim"], case["context"]
    inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv
    ang = torch.cat([ang, ang], dim=-1)
    return ang.cos().float(), ang.sin().float()


def _inputs(case, seed):
    """Every tensor of the call, dense: activations [batch, tokens, heads, d]."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 2654435761 % (1 << 62))
    dt, b, t, d = _dtype(case), case["batch"], case["tokens"], case["head_dim"]
    s = {}
    if case["kind"] != "append" or case["rotate"]:
        s["q"] = _randn(gen, b, t, case["heads"], d).to(dt)
    if case["kind"] != "decode":
        s["k"] = _randn(gen, b, t, case["kv_heads"], d).to(dt)
        s["v"] = _randn(gen, b, t, case["kv_heads"], d).to(dt)
    if case["kind"] == "window":
        if case["train"]:
            s["dy"] = _randn(gen, b, t, case["heads"], d).to(dt)
        return s
    each = _pages_each(case)
    pages = (b * each, case["kv_heads"], case["page"], d)
    s["table"] = torch.randperm(b * each, generator=gen, device="cuda").int().view(b, each)
    starts, counts = _lengths(case)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
    if case["bits"] == 4:
        s["k_pages"], s["k_scales"] = _packed(gen, pages)
        s["v_pages"], s["v_scales"] = _packed(gen, pages)
    else:
        s["k_pages"], s["v_pages"] = _randn(gen, *pages).to(dt), _randn(gen, *pages).to(dt)
    if case.get("rotate"):
        s["cos"], s["sin"] = _tables(case)
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
    if own:
        pkg = str(Path(__file__).resolve().parents[1] / "torch-mojo-backend_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from torch_mojo_backend import register_mojo_devices
        from torch_mojo_backend.kv_cache import PagedKVCache

        register_mojo_devices()
        s = {n: _mojo(t) for n, t in s.items()}
        if case["kind"] != "window":
            s["cache"] = PagedKVCache(s["k_pages"], s["v_pages"], s.get("k_scales"), s.get("v_scales"))
    # heads in front, as views of a projection's output
    for n in ("q", "k", "v", "dy"):
        if n in s:
            s[n] = s[n].transpose(1, 2)
    if own and case["kind"] == "window" and case["train"]:
        for n in ("q", "k", "v"):
            s[n].requires_grad_()
    s["case"] = dict(case)
    return s


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"append": _own_append, "decode": _own_decode, "window": _own_window}[kind](s)
    return {"append": _append, "decode": _decode, "window": _window}[kind](s)


def _own_append(s):
    from torch_mojo_backend import ops

    q = ops.paged_append(s["cache"], s["table"], s["starts"], s["k"], s["v"], s.get("cos"), s.get("sin"),
                         q=s.get("q"), counts=s["counts"])
    if s["case"]["bits"] == 4:
        k, v = ops.paged_gather(s["cache"], s["table"], s["starts"], s["case"]["tokens"], counts=s["counts"],
                                dtype=torch.float32)
        return {"q": q, "k": k, "v": v}
    return {"q": q, "k": s["k_pages"], "v": s["v_pages"]}


def _own_decode(s):
    from torch_mojo_backend import ops

    c = s["case"]
    return ops.paged_attention(s["q"], s["cache"], s["table"], s["starts"], counts=s["counts"], window=c["window"],
                               sinks=c["sinks"])


def _own_window(s):
    from torch_mojo_backend import ops

    c = s["case"]
    if not c["train"]:
        with torch.no_grad():
            return ops.sliding_window_attention(s["q"], s["k"], s["v"], c["window"], sinks=c["sinks"])
    for n in ("q", "k", "v"):
        s[n].grad = None
    out = ops.sliding_window_attention(s["q"], s["k"], s["v"], c["window"], sinks=c["sinks"])
    out.backward(s["dy"])
    return {"out": out.detach(), "dq": s["q"].grad, "dk": s["k"].grad, "dv": s["v"].grad}


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------
def _unpack(codes, scales):
    """f32 values of 4-bit rows.  A row's 32-bit words hold eight channels
    each: word g * (d / 32) + s the channels 32 s + 8 g .. + 7, even ones in
    the low 16 bits."""
    *lead, half = codes.shape
    n = half // 16
    x = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(*lead, 4, n, 2, 4)
    x = x.transpose(-1, -2).transpose(-4, -3).reshape(*lead, n, GROUP).float()
    scales = scales.float()
    return (scales[..., 1:] + scales[..., :1] * x).flatten(-2)


def _pack(x):
    """(codes, scales) of f64 rows."""
    *lead, d = x.shape
    n = d // GROUP
    x = x.clamp(-LIMIT, LIMIT).reshape(*lead, n, GROUP)
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scales = torch.cat([(high - low) / 15.0, low], dim=-1).float().half()
    step, base = scales[..., :1].double(), scales[..., 1:].double()
    codes = torch.where(step > 0, ((x - base) / torch.where(step > 0, step, 1.0)).round().clamp(0, 15), 0.0)
    words = codes.to(torch.uint8).reshape(*lead, n, 4, 4, 2).transpose(-1, -2).transpose(-4, -3)
    words = words.reshape(*lead, 4 * n * 4, 2)
    return words[..., 0] | (words[..., 1] << 4), scales


def _rotated(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], dim=-1) * sin


def _places(s, tokens):
    """position, whether it is a token, its page and its slot [batch, tokens]."""
    page = s["case"]["page"]
    t = torch.arange(tokens, device="cuda")
    pos = s["starts"].long()[:, None] + t
    real = t < s["counts"][:, None]
    at = torch.where(real, pos, 0)
    return at, real, s["table"].long().gather(1, at // page), at % page


def _append(s):
    c = s["case"]
    four = c["bits"] == 4
    at, real, page, slot = _places(s, c["tokens"])
    wide = torch.float64 if four else torch.float32  # a code next to a border turns on the last bit
    k, v, q = s["k"].transpose(1, 2), s["v"].transpose(1, 2), None
    if c["rotate"]:
        q = s["q"].transpose(1, 2)
        cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
        q = torch.where(real[:, :, None, None], _rotated(q.float(), cos, sin), 0.0).to(q.dtype).transpose(1, 2)
        k = _rotated(k.to(wide), cos.to(wide), sin.to(wide))
    rows = (page[real], slice(None), slot[real])
    if not four:
        s["k_pages"][rows], s["v_pages"][rows] = k[real].to(s["k_pages"].dtype), v[real].to(s["v_pages"].dtype)
        return {"q": q, "k": s["k_pages"], "v": s["v_pages"]}
    for n, x in (("k", k), ("v", v)):
        s[n + "_pages"][rows], s[n + "_scales"][rows] = _pack(x[real].double())
    back = [torch.where(real[:, :, None, None], _unpack(s[n + "_pages"][page, :, slot], s[n + "_scales"][page, :, slot]),
                        0.0).transpose(1, 2) for n in ("k", "v")]
    return {"q": q, "k": back[0], "v": back[1]}


def _visible(pos, keys, window, sinks):
    """Whether the query at pos [..., t] sees key j: [..., t, keys]."""
    j = torch.arange(keys, device="cuda")
    pos = pos[..., None]
    keep = j <= pos
    return keep & ((pos - j < window) | (j < sinks)) if window else keep


def _softmax(scores, keep):
    """exp(scores) over the kept keys, normalised; zero where none is kept."""
    scores = scores.masked_fill(~keep, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0)


def _decode(s):
    c = s["case"]
    table = s["table"].long()
    b, d, hk = c["batch"], c["head_dim"], c["kv_heads"]

    def rows(n):
        if c["bits"] == 4:
            x = _unpack(s[n + "_pages"][table], s[n + "_scales"][table])
        else:
            x = s[n + "_pages"][table].float()
        return x.transpose(1, 2).reshape(b, hk, -1, d)

    k, v = rows("k"), rows("v")
    t = torch.arange(c["tokens"], device="cuda")
    pos = torch.where(t < s["counts"][:, None], s["starts"][:, None] + t, -1)
    keep = _visible(pos, k.shape[2], c["window"], c["sinks"])[:, None, None]
    q = s["q"].float().reshape(b, hk, -1, d)
    p = _softmax((q @ k.transpose(-1, -2)).view(b, hk, -1, c["tokens"], k.shape[2]) / math.sqrt(d), keep)
    seen = keep.any(3)[:, :, 0, :, None]  # what lies in pages behind the last token is no number to count on
    out = p.view(b, hk, -1, k.shape[2]) @ torch.where(seen, v, 0.0)
    return out.view(b, c["heads"], c["tokens"], d).to(s["q"].dtype)


def _window(s):
    c = s["case"]
    b, t, d, hk = c["batch"], c["tokens"], c["head_dim"], c["kv_heads"]
    q = s["q"].float().reshape(b, hk, -1, t, d)
    k, v = s["k"].float()[:, :, None], s["v"].float()[:, :, None]
    scale = 1.0 / math.sqrt(d)
    keep = _visible(torch.arange(t, device="cuda"), t, c["window"], c["sinks"])
    p = _softmax((q @ k.transpose(-1, -2)).mul_(scale), keep)
    out = p @ v
    dt = s["q"].dtype
    if not c["train"]:
        return out.view(b, -1, t, d).to(dt)
    dy = s["dy"].float().reshape(q.shape)
    dv = (p.transpose(-1, -2) @ dy).sum(2)
    ds = (dy @ v.transpose(-1, -2)).sub_((dy * out).sum(-1, keepdim=True)).mul_(p)
    dq = (ds @ k).mul_(scale)
    dk = (ds.transpose(-1, -2) @ q).sum(2).mul_(scale)
    return {"out": out.view(b, -1, t, d).to(dt), "dq": dq.view(b, -1, t, d).to(dt), "dk": dk.to(dt), "dv": dv.to(dt)}


# ---------------------------------------------------------------------------
# what one call cannot do without
# ---------------------------------------------------------------------------
def _seen(pos, window, sinks):
    """How many keys the query at pos sees."""
    near = min(pos + 1, window) if window else pos + 1
    return near + (min(sinks, pos + 1 - near) if window else 0)


def work(case):
    d, h, hk = case["head_dim"], case["heads"], case["kv_heads"]
    e = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "window":
        rows = case["batch"] * case["tokens"]
        pairs = case["batch"] * h * sum(_seen(i, case["window"], case["sinks"]) for i in range(case["tokens"]))
        own_rows, shared = rows * h * d * e, rows * hk * d * e
        if case["train"]:  # q, k, v, dO in; O, dQ, dK, dV out
            return {"bytes": 4 * own_rows + 4 * shared, "flops": 14.0 * d * pairs}
        return {"bytes": 2 * own_rows + 2 * shared, "flops": 4.0 * d * pairs}
    row = d // 2 + d // 8 if case["bits"] == 4 else d * e  # of the cache, one head
    starts, counts = _lengths(case)
    n = sum(counts)
    if case["kind"] == "append":
        moved = 2 * n * hk * (d * e + row)
        if case["rotate"]:
            moved += 2 * n * h * d * e + 8 * d * min(n, case["context"])
        if case["bits"] == 4:  # and read back as f32 values
            moved += 2 * n * hk * (row + 4 * d)
        return {"bytes": moved, "flops": (3.0 * n * d * (h + hk) if case["rotate"] else 0.0)}
    pairs = read = 0
    for s, c in zip(starts, counts):
        if not c:
            continue
        pairs += sum(_seen(s + t, case["window"], case["sinks"]) for t in range(c))
        last = s + c - 1
        near = min(last + 1, case["window"] + c - 1) if case["window"] else last + 1
        read += near + (min(case["sinks"], last + 1 - near) if case["window"] else 0)
    return {"bytes": 2 * read * hk * row + 2 * n * h * d * e, "flops": 4.0 * d * h * pairs}


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_values(codes, scales, d):
    """f64 values of 4-bit rows, channel by channel."""
    c = torch.arange(d, device="cuda")
    word = (c % 32) // 8 * (d // 32) + c // 32
    nibble = (c % 8) // 2 + 4 * (c % 2)
    byte = codes[..., 4 * word + nibble // 2].long()
    code = (byte >> (4 * (nibble % 2))) & 15
    pair = scales.double()[..., c // GROUP, :]
    return pair[..., 1] + pair[..., 0] * code


def _exact_turn(x, cos, sin):
    """x [tokens, heads, d] turned by the angles of its tokens."""
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    c, s = cos.double()[:, None], sin.double()[:, None]
    return torch.cat([a * c[..., :half] - b * s[..., :half], b * c[..., half:] + a * s[..., half:]], dim=-1)


def _exact_append(case, s):
    starts, counts = _lengths(case)
    d, four = case["head_dim"], case["bits"] == 4
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda") if case["rotate"] else None
    if four:
        k = torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda")
        v = torch.zeros_like(k)
    else:
        k, v = s["k_pages"].double(), s["v_pages"].double()
    for b, (start, n) in enumerate(zip(starts, counts)):
        if not n:
            continue
        new = {x: s[x][b, :n].double() for x in ("q", "k", "v") if x in s}
        at = torch.arange(start, start + n, device="cuda")
        if case["rotate"]:
            for x in ("q", "k"):
                new[x] = _exact_turn(new[x], s["cos"][at], s["sin"][at])
            q[b, :n] = new["q"]
        for whole, x in ((k, new["k"]), (v, new["v"])):
            if four:
                g = x.clamp(-LIMIT, LIMIT).unflatten(-1, (-1, GROUP))
                low = g.min(-1, keepdim=True).values
                step = ((g.max(-1, keepdim=True).values - low) / 15).float().half().double()
                low = low.float().half().double()
                code = torch.nan_to_num((g - low) / step).round().clamp(0, 15)
                whole[b, :n] = (low + step * code).flatten(-2)
            else:
                whole[s["table"][b].long()[at // case["page"]], :, at % case["page"]] = x
    if case["rotate"]:
        q = q.transpose(1, 2)
    if four:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    return {"q": q, "k": k, "v": v}


def _exact_decode(case, s):
    starts, counts = _lengths(case)
    d, g = case["head_dim"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (start, n) in enumerate(zip(starts, counts)):
        if not n:
            continue
        j = torch.arange(start + n, device="cuda")
        page, slot = s["table"][b].long()[j // case["page"]], j % case["page"]
        pos = torch.arange(start, start + n, device="cuda")[:, None]
        hidden = j > pos
        if case["window"]:
            hidden |= (pos - j >= case["window"]) & (j >= case["sinks"])
        for h in range(case["kv_heads"]):
            if case["bits"] == 4:
                k, v = (_exact_values(s[x + "_pages"][page, h, slot], s[x + "_scales"][page, h, slot], d) for x in "kv")
            else:
                k, v = (s[x + "_pages"][page, h, slot].double() for x in "kv")
            q = s["q"][b, :n, h * g:(h + 1) * g].double().transpose(0, 1)
            w = torch.softmax(((q @ k.T) / math.sqrt(d)).masked_fill(hidden, -math.inf), dim=-1)
            out[b, :n, h * g:(h + 1) * g] = (w @ v).transpose(0, 1)
    return out.transpose(1, 2)


def _exact_window(case, s):
    t, d, g = case["tokens"], case["head_dim"], case["heads"] // case["kv_heads"]
    i = torch.arange(t, device="cuda")[:, None]
    j = i.T
    hidden = (j > i) | ((i - j >= case["window"]) & (j >= case["sinks"]))
    got = {n: torch.zeros(s[x].shape, dtype=torch.float64, device="cuda")
           for n, x in (("out", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v"))}
    for b in range(case["batch"]):
        for h in range(case["heads"]):
            q, k, v = (s[x][b, :, y].double().requires_grad_() for x, y in (("q", h), ("k", h // g), ("v", h // g)))
            w = torch.softmax(((q @ k.T) / math.sqrt(d)).masked_fill(hidden, -math.inf), dim=-1)
            out = w @ v
            got["out"][b, :, h] = out.detach()
            if case["train"]:
                dq, dk, dv = torch.autograd.grad(out, (q, k, v), s["dy"][b, :, h].double())
                got["dq"][b, :, h] = dq
                got["dk"][b, :, h // g] += dk
                got["dv"][b, :, h // g] += dv
    got = {n: x.transpose(1, 2) for n, x in got.items()}
    return got if case["train"] else got["out"]


def exact(case, seed):
    s = _inputs(case, seed)
    return {"append": _exact_append, "decode": _exact_decode, "window": _exact_window}[case["kind"]](case, s)
