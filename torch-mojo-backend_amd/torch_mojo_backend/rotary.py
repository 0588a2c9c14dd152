"""Frequencies of rotary positions, also for contexts longer than those that a
model was trained on."""

from __future__ import annotations

import math
from typing import NamedTuple

import torch


class RotaryFrequencies(NamedTuple):
    """Radians a position of each pair of channels (f64), and what the turned
    channels are multiplied with; both go to `ops.rotary_at`."""

    frequencies: torch.Tensor
    scale: float


def rotary_frequencies(turned, base=10000.0, *, scaling=None, factor=1.0, length=None, slow=1.0, fast=32.0, device="mojo"):
    """base ** (-2 j / turned) for the pairs j of `turned` channels, changed by
    `scaling` for a context `factor` times as long as the trained one:

    - "linear": every frequency divided by factor (positions interpolated);
    - "base": a larger base, base * factor ** (turned / (turned - 2)), which leaves
      the fastest pair as it is and divides the slowest frequency by factor;
    - "parts": by part of the spectrum (YaRN, Peng et al. 2023): pairs of fewer than
      `slow` turns over the trained `length` are divided by factor, those of more
      than `fast` are not, pairs between by a linear mix over their number; the
      turned channels are multiplied with 0.1 ln(factor) + 1."""
    turned = int(turned)
    if turned <= 0 or turned % 2:
        raise ValueError(f"rotary_frequencies: {turned} channels to turn, expected an even number")
    base, factor = float(base), float(factor)
    if not base > 1.0 or not math.isfinite(base) or not factor >= 1.0 or not math.isfinite(factor):
        raise ValueError(f"rotary_frequencies: base {base} must be above 1, factor {factor} at least 1")
    j = torch.arange(0, turned, 2, dtype=torch.float64)
    scale = 1.0
    if scaling == "base":
        if turned < 4:
            raise ValueError("rotary_frequencies: scaling 'base' needs two pairs or more")
        base *= factor ** (turned / (turned - 2))
    freq = base ** (-j / turned)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "parts":
        if length is None or not length > 0 or not fast > slow > 0:
            raise ValueError(f"rotary_frequencies: scaling 'parts' needs the trained length, got {length}, and slow {slow} < fast {fast}")
        # the pair of a given number of turns over the length, as a real number
        pair = lambda turns: turned * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), turned - 1)
        divided = ((j / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq * (1 - divided) + freq / factor * divided
        scale = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "base"):
        raise ValueError(f"rotary_frequencies: scaling {scaling!r} (linear, base or parts)")
    return RotaryFrequencies(freq.to(device), scale)


def turn_plain(x, positions, frequencies, interleaved, scale, inverse=False):
    """The plain formula of `ops.rotary_at` for x [batch, heads, tokens, d]."""
    n = 2 * frequencies.shape[0]
    wide = torch.promote_types(x.dtype, torch.float32)
    angle = positions.double()[..., None, :, None] * frequencies
    cos, sin = (angle.cos() * scale).to(wide), (angle.sin() * (-scale if inverse else scale)).to(wide)
    a, rest = x[..., :n].to(wide), x[..., n:]
    if interleaved:
        even, odd = a[..., 0::2], a[..., 1::2]
        a = torch.stack([even * cos - odd * sin, odd * cos + even * sin], dim=-1).flatten(-2)
    else:
        low, high = a[..., :n // 2], a[..., n // 2:]
        a = torch.cat([low * cos - high * sin, high * cos + low * sin], dim=-1)
    return torch.cat([a.to(x.dtype), rest], dim=-1)
