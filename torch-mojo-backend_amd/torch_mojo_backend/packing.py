"""Sequences of different lengths, packed: their rows laid end to end, without
padding between them.

A `PackedSequences` says where each one begins.  It is made once for a batch
and serves all of a model's layers: `ops.packed_attention` keeps every row to
its own sequence, `positions` are the rows' positions for `ops.rotary_at` or an
embedding.  On the mojo device making it runs two small kernels that lay out
the attention's work; elsewhere the plain formulas below run (the CPU
reference).
"""

from __future__ import annotations

import itertools
import math

import torch

from .mojo_device.torch_mojo_tensor import TorchMojoTensor

_MOST = 2 ** 30 - 1024  # rows of a batch


class PackedSequences:
    """Sequence i is rows offsets[i] .. offsets[i + 1] - 1 of `tokens` rows:
    offsets is int32 [sequences + 1], rising from 0 on, or from further on, up to
    tokens at most.  Sequences may be empty; rows before the first and behind the
    last one belong to none.

    `positions` int32 [tokens] are the rows' places in their sequences (0 of
    rows without one).  The offsets are read when this is made, and changes to
    the tensor afterwards are not seen.  Offsets that fall or leave the rows
    raise IndexError, on the mojo device at the next device-to-host read; all
    rows then belong to none."""

    def __init__(self, offsets, tokens):
        tokens = int(tokens)
        if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.shape[0] < 1:
            raise ValueError(f"PackedSequences: offsets must be int32 [sequences + 1], got {tuple(offsets.shape)}"
                             f" of {offsets.dtype}")
        if not 0 <= tokens < _MOST or offsets.shape[0] > _MOST:
            raise ValueError(f"PackedSequences: {offsets.shape[0] - 1} sequences of {tokens} rows (fewer than {_MOST})")
        self.tokens, self.count, self.device = tokens, offsets.shape[0] - 1, offsets.device
        self.on_mojo = isinstance(offsets, TorchMojoTensor)
        if self.on_mojo:
            from .eager_kernels import packed

            self._plan, self.positions = packed.plan(offsets, tokens)
            return
        self._offsets = at = offsets.tolist()
        if at[0] < 0 or at[-1] > tokens or any(b < a for a, b in itertools.pairwise(at)):
            raise IndexError("offsets of packed sequences fall or leave the rows")
        self.positions = torch.zeros(tokens, dtype=torch.int32, device=offsets.device)
        for a, b in itertools.pairwise(at):
            self.positions[a:b] = torch.arange(b - a, dtype=torch.int32, device=offsets.device)

    @classmethod
    def of_lengths(cls, lengths, tokens=None, *, device="mojo"):
        """Sequences of these lengths from row 0 on, of `tokens` rows (default:
        no more than theirs)."""
        lengths = [int(n) for n in lengths]
        if any(n < 0 for n in lengths):
            raise ValueError(f"PackedSequences: lengths must not be negative, got {min(lengths)}")
        total = sum(lengths)
        tokens = total if tokens is None else int(tokens)
        if total > tokens:
            raise ValueError(f"PackedSequences: {total} rows of sequences in {tokens}")
        if not tokens < _MOST:
            raise ValueError(f"PackedSequences: {tokens} rows (fewer than {_MOST})")
        at = [0, *itertools.accumulate(lengths)]
        return cls(torch.tensor(at, dtype=torch.int32).to(device), tokens)


    def next_tokens(self, tokens, ignore_index=-100):
        """For each row of tokens [tokens] the token behind it in its sequence,
        ignore_index where there is none: what a model's row predicts."""
        if tokens.dim() != 1 or tokens.shape[0] != self.tokens:
            raise ValueError(f"PackedSequences: tokens must be [{self.tokens}], got {tuple(tokens.shape)}")
        if not self.tokens:
            return tokens.clone()
        # (a row whose position is 0 begins a sequence, or belongs to none)
        behind = torch.where(self.positions[1:] > 0, tokens[1:], torch.full_like(tokens[1:], ignore_index))
        return torch.cat([behind, torch.full_like(tokens[:1], ignore_index)])


def nothing_of(q, k, v):
    """The result of empty q, k and v, whose gradients are there all the same."""
    return q + (k.sum() + v.sum())


def attention_plain(q, k, v, sequences, window, scale):
    """The plain formula of `ops.packed_attention`, in 32 bits at least."""
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else scale
    wide = torch.promote_types(q.dtype, torch.float32)
    at, group = sequences._offsets, q.shape[1] // k.shape[1]
    parts = [nothing_of(q[:0], k[:0], v[:0]), torch.zeros_like(q[:at[0]])]
    for a, b in itertools.pairwise(at):
        if a == b:
            continue
        i = torch.arange(b - a, device=q.device)
        hidden = i[None, :] > i[:, None]
        if window:
            hidden = hidden | (i[:, None] - i[None, :] >= window)
        qs = q[a:b].to(wide).transpose(0, 1)
        ks, vs = (x[a:b].to(wide).transpose(0, 1).repeat_interleave(group, 0) for x in (k, v))
        p = torch.softmax((qs @ ks.transpose(-1, -2) * scale).masked_fill(hidden, -math.inf), dim=-1)
        parts.append((p @ vs).transpose(0, 1).to(q.dtype))
    return torch.cat([*parts, torch.zeros_like(q[at[-1]:])])
