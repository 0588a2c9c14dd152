"""Inputs and f64 results for the tests of the paged cache, on any device."""

from __future__ import annotations

import numpy as np
import torch

from oracle import paged as oracle
from torch_mojo_backend.kv_cache import PagedKVCache

STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative


def np64(t):
    return t.detach().cpu().double().numpy()


class Case:
    """A cache of `lengths` tokens per sequence, pages in random order, whose
    slots that no sequence owns hold NaN."""

    def __init__(self, lengths, *, hk=2, d=64, page=16, dtype=torch.bfloat16, bits=None, device="cpu", seed=0,
                 spare=3, slots_first=False, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.hk, self.d, self.page, self.device = list(lengths), hk, d, page, device
        b = len(self.lengths)
        self.width = max(1, max((-(-n // page) for n in self.lengths), default=0))
        total = b * self.width + spare
        order = torch.randperm(total, generator=g)[:b * self.width].view(b, self.width)
        self.table = order.int()
        rows = [spread * torch.randn(b, hk, self.width * page, d, generator=g) for _ in range(2)]
        self.bits, self.dtype = bits, dtype
        shape = (total, page, hk) if slots_first else (total, hk, page)
        tensors = []
        self.values = []
        for x in rows:
            if bits == 4:
                codes, scale, low = oracle.quantize(x.double().numpy())
                self.values.append(oracle.values(codes, scale, low))
                at = [oracle.place_of(c, d) for c in range(d)]
                packed = np.zeros((*codes.shape[:-1], d // 2), dtype=np.uint8)
                for c, (byte, nibble) in enumerate(at):
                    packed[..., byte] |= (codes[..., c] << (4 * nibble)).astype(np.uint8)
                pages = torch.full((*shape, d // 2), 0xA5, dtype=torch.uint8)
                scales = torch.full((*shape, d // 32, 2), float("nan"), dtype=torch.float16)
                pair = torch.from_numpy(np.stack([scale, low], -1))
                self._fill(pages, torch.from_numpy(packed), slots_first)
                self._fill(scales, pair, slots_first)
                tensors.append((pages, scales))
            else:
                x = x.to(dtype)
                self.values.append(x.double().numpy())
                pages = torch.full((*shape, d), float("nan"), dtype=dtype)
                self._fill(pages, x, slots_first)
                tensors.append((pages, None))
        put = (lambda t: t.to(device).transpose(1, 2)) if slots_first else (lambda t: t.to(device))
        (k, ks), (v, vs) = tensors
        self.cache = PagedKVCache(put(k), put(v), put(ks) if ks is not None else None, put(vs) if vs is not None else None)
        self.dev_table = self.table.to(device)

    def _fill(self, pages, x, slots_first):
        for b, n in enumerate(self.lengths):
            for j in range(n):
                p, s = int(self.table[b, j // self.page]), j % self.page
                pages[(p, s) if slots_first else (p, slice(None), s)] = x[b, :, j]

    def ints(self, v):
        return torch.tensor(v, dtype=torch.int32).to(self.device)

    def queries(self, h, t, dtype=None, seed=1):
        g = torch.Generator().manual_seed(seed)
        return torch.randn(len(self.lengths), h, t, self.d, generator=g).to(dtype or self.dtype)

    def expected(self, q, starts, counts, window=0, sinks=0, scale=None):
        """(o, bound): the f64 result and how far a result in q's dtype may be
        off.  Rounding the result: half a step.  Sums in f32 of n products:
        n + 8 roundings of 2^-24 of the absolute sum.  4-bit rows are rounded
        once to f16 (2^-11), as are the weights, where 16-bit products use
        them; an error ds of the scores changes o by at most 2 ds max|v| (1 +
        2 ds)."""
        b, h, t, d = q.shape
        qn, out, bound = np64(q), np.zeros(q.shape), np.zeros(q.shape)
        sc = d ** -0.5 if scale is None else scale
        for i in range(b):
            n = starts[i] + min(counts[i], t)
            if counts[i] <= 0:
                continue
            k, v = (x[i][:, :n] for x in self.values)
            pos = [starts[i] + u if u < counts[i] else -1 for u in range(t)]
            out[i] = oracle.attend(qn[i], k, v, pos, window, sinks, scale)
            size = abs(sc) * (np.abs(np.repeat(k, h // self.hk, 0)) @ np.abs(qn[i]).swapaxes(-1, -2)).max()
            ds = size * ((d + 8) * 2.0 ** -24 + (2.0 ** -11 if self.bits == 4 else 0))
            top = np.abs(v).max()
            bound[i] = top * (2 * ds * (1 + 2 * ds) + (n + 8) * 2.0 ** -24 + (2 * 2.0 ** -11 if self.bits == 4 else 2.0 ** -15))
            bound[i][:, [p < 0 for p in pos]] = 0.0
        return out, bound + STEP[q.dtype] * np.abs(out)


def check(actual, expected, bound, what=""):
    a = np64(actual)
    assert a.shape == expected.shape, (what, a.shape, expected.shape)
    bad = ~(np.abs(a - expected) <= bound)
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} off; first at {i}: got {a[i]}, expected {expected[i]}"
                             f" +- {bound[i]}; largest ratio {np.nanmax(np.abs(a - expected) / np.maximum(bound, 1e-300)):.3g}")
