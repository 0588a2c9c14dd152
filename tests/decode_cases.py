"""Token-by-token runs of a small Gemma-3-shaped model, on any device."""

from __future__ import annotations

import torch

from torch_mojo_backend.gemma3 import Gemma3, Gemma3Config


def model(dtype, device, *, head_dim=64, window=7, sinks=2, hidden=64):
    """(model on the device, the same rounded weights in f64 on the CPU)."""
    cfg = Gemma3Config(vocab_size=97, hidden=hidden, layers=3, heads=4, kv_heads=2, head_dim=head_dim, d_ff=96,
                       window=window, sinks=sinks, global_every=3)
    torch.manual_seed(0)
    ref = Gemma3(cfg)
    for _, p in ref.named_parameters():
        if p.dim() == 1:
            torch.nn.init.normal_(p, std=0.1)
    ref = ref.to(dtype)
    m = Gemma3(cfg)
    m.load_state_dict(ref.state_dict())
    return m.to(dtype).to(device), ref.double()


def tokens(batch, length):
    return torch.randint(0, 97, (batch, length), generator=torch.Generator().manual_seed(1))


def run(m, idx, steps, device, *, page=4, bits=None):
    """Logits [B, T, vocab] of idx [B, T], fed by calls of steps: each a list
    of how many tokens a sequence takes (the most of them is the call's T)."""
    b, t = idx.shape
    width = -(-t // page)
    order = torch.randperm(b * width + 2, generator=torch.Generator().manual_seed(2))[:b * width]
    table = order.view(b, width).int().to(device)
    caches = m.caches(b * width + 2, page, bits=bits)
    out = torch.full((b, t, 97), float("nan"), dtype=torch.float64)
    at = [0] * b
    for counts in steps:
        n = max(counts)
        part = torch.zeros(b, n, dtype=torch.int64)
        for i, c in enumerate(counts):
            part[i, :c] = idx[i, at[i]:at[i] + c]
        ints = lambda x: torch.tensor(x, dtype=torch.int32).to(device)  # noqa: E731
        got = m.forward_cached(part.to(device), caches, table, ints(at), None if min(counts) == n else ints(counts))
        got = got.cpu().double()
        for i, c in enumerate(counts):
            out[i, at[i]:at[i] + c] = got[i, :c]
            at[i] += c
    assert at == [t] * b
    return out


def bound(dtype, want, width):
    """How far logits of three layers may be off: each layer has four products
    of sums (up to `width` terms, f32) one after another, its two attention
    products, five norms, the rotation, the activation and two additions, and
    each result is rounded to the type: 14 roundings a layer, 2 more at the
    ends, of half a step, and (width + 8) steps of f32 in each of the 7 sums.
    Norms keep relative errors; the largest logit is the measure."""
    half = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}[dtype]
    return ((3 * 14 + 2) * half + 22 * (width + 8) * 2.0 ** -24) * want.abs().max().item()
