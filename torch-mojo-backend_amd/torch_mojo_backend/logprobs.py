"""Log-probabilities of given tokens: what `ops.token_logprobs` returns, and its
plain formula."""

from __future__ import annotations

from typing import NamedTuple

import torch


class TokenLogprobs(NamedTuple):
    """Of each row: the given token's log-probability (None without tokens), the
    entropy in nats, and the largest entries' log-probabilities and tokens, largest
    first (None where not asked for)."""

    logprobs: torch.Tensor | None
    entropy: torch.Tensor | None
    top_logprobs: torch.Tensor | None
    top_tokens: torch.Tensor | None


def plain(logits, tokens, top, entropy, ignore_index):
    x = logits.to(torch.promote_types(logits.dtype, torch.float32))
    logp = torch.log_softmax(x, dim=-1)
    picked = best = order = spread = None
    if tokens is not None:
        ignored = tokens == ignore_index
        if (((tokens < 0) | (tokens >= x.shape[-1])) & ~ignored).any():
            raise IndexError("Target is out of bounds")
        picked = logp.gather(-1, tokens.masked_fill(ignored, 0)[..., None])[..., 0].masked_fill(ignored, 0.0)
    if entropy:  # (what has no probability adds nothing)
        spread = -(torch.exp(logp) * logp.clamp(min=-1e4)).sum(-1)
    if top:
        order = torch.sort(x.detach(), dim=-1, descending=True, stable=True)[1][..., :top]
        best = logp.gather(-1, order)
    return TokenLogprobs(picked, spread, best, order)
