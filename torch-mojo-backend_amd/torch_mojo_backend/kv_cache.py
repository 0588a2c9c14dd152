"""Keys and values of earlier tokens, held in pages.

A `PagedKVCache` is the storage of one attention layer: a page holds
`page_size` tokens of every K/V head, and a page table [batch, pages] says
which pages a sequence owns, in order, so sequences of different lengths share
one allocation and grow a page at a time.  `torch_mojo_backend.ops` has the
operations on it: `paged_append`, `paged_attention`, `paged_gather`.  They run
one gfx950 kernel each on the mojo device (attention a second one, where blocks
share the keys of a row) and the plain formulas below elsewhere (the CPU
reference).

With `bits=4` a row of `head_dim` channels is held as 4-bit codes with a scale
and a minimum in float16 for each 32 channels (5 bits a value): minimum =
min, scale = (max - min) / 15, value = minimum + scale * code.  Inputs are
clamped to +-61440; 32 channels with a NaN or an infinity among them read back
as NaN.  Attention takes such values in float16: pages that were not filled by
`paged_append` must keep to its range, minimum + scale * code within +-65504 and
scale from 0 to 8192, or their values may become infinities and NaN there.
"""

from __future__ import annotations

import torch

from .mojo_device.torch_mojo_tensor import TorchMojoTensor

GROUP = 32  # channels that share a scale and a minimum in a 4-bit cache
_LIMIT = 61440.0
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


class PagedKVCache:
    """Pages of keys and values: k, v [num_pages, kv_heads, page_size,
    head_dim] of a float dtype, or, with k_scales and v_scales [num_pages,
    kv_heads, page_size, head_dim / 32, 2] in float16, uint8 codes
    [num_pages, kv_heads, page_size, head_dim / 2].  The tensors are those it
    was made with; a copy of the cache is made from copies of them."""

    def __init__(self, k, v, k_scales=None, v_scales=None):
        for name, t in (("k", k), ("v", v)):
            if t.dim() != 4 or t.shape != k.shape or t.dtype != k.dtype or t.device != k.device:
                raise ValueError(f"PagedKVCache: k and v must be alike, [pages, kv_heads, page_size, head_dim];"
                                 f" {name} is {tuple(t.shape)} of {t.dtype} on {t.device}")
        if (k_scales is None) != (v_scales is None):
            raise ValueError("PagedKVCache: k_scales and v_scales come together")
        self.num_pages, self.kv_heads, self.page_size, width = k.shape
        if k_scales is None:
            self.bits, self.head_dim, self.dtype = 8 * k.dtype.itemsize, width, k.dtype
            if k.dtype not in _FLOATS:
                raise TypeError(f"PagedKVCache: pages of {k.dtype} are not supported without scales")
        else:
            self.bits, self.head_dim, self.dtype = 4, 2 * width, torch.uint8
            if k.dtype != torch.uint8:
                raise TypeError(f"PagedKVCache: 4-bit codes must be uint8, not {k.dtype}")
        if self.head_dim % (8 if k_scales is None else GROUP) or not 0 < self.head_dim <= 256:
            raise ValueError(f"PagedKVCache: head_dim {self.head_dim} must be a multiple of"
                             f" {8 if k_scales is None else GROUP} up to 256")
        if min(k.shape) <= 0:
            raise ValueError(f"PagedKVCache: empty pages {tuple(k.shape)}")
        if k_scales is not None:
            want = (*k.shape[:3], self.head_dim // GROUP, 2)
            for t in (k_scales, v_scales):
                if tuple(t.shape) != want or t.dtype != torch.float16 or t.device != k.device:
                    raise ValueError(f"PagedKVCache: scales must be float16 {want} on {k.device}, got"
                                     f" {tuple(t.shape)} of {t.dtype} on {t.device}")
                if t.stride()[3:] != (2, 1):
                    raise ValueError("PagedKVCache: the pairs of a row of scales must be contiguous")
        tensors = [t for t in (k, v, k_scales, v_scales) if t is not None]
        for t in tensors:
            if t.requires_grad:
                raise ValueError("PagedKVCache: pages hold values without gradients")
            if t.stride(-1) != 1:
                raise ValueError("PagedKVCache: rows of pages must be contiguous")
            if _overlaps(t):
                raise ValueError("PagedKVCache: rows of pages must not overlap")
        if any(_share(a, b) for i, a in enumerate(tensors) for b in tensors[:i]):
            raise ValueError("PagedKVCache: pages of keys, of values and scales must not share memory")
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales
        self.tensors = tuple(tensors)
        self.scale = self.head_dim ** -0.5  # attention's default
        self.on_mojo = all(isinstance(t, TorchMojoTensor) for t in tensors)
        if self.on_mojo:
            for t in (k, v):
                if t._ptr % 16 or any(s * t._itemsize % 16 for s in t._strides[:3]):
                    raise ValueError("PagedKVCache: rows of pages must be 16-byte aligned")
            if k_scales is not None and any(t._ptr % 4 or any(s % 2 for s in t._strides[:3])
                                            for t in (k_scales, v_scales)):
                raise ValueError("PagedKVCache: rows of scales must be 4-byte aligned")
            from .eager_kernels import paged

            self._desc = paged.describe(self)
            self.holders = frozenset(id(t._holder) for t in tensors)  # their storages, which live as long as the cache

    def __setattr__(self, name, value):
        # the kernels go by the addresses of the tensors that the cache was made with
        if name in ("k", "v", "k_scales", "v_scales") and name in self.__dict__:
            raise AttributeError(f"PagedKVCache: {name} is fixed: copy into it, or make another cache")
        super().__setattr__(name, value)

    def __reduce__(self):  # the kernels' description holds addresses
        return type(self), (self.k, self.v, self.k_scales, self.v_scales)

    @property
    def device(self):
        return self.k.device

    @classmethod
    def zeros(cls, num_pages, page_size, kv_heads, head_dim, *, dtype=torch.bfloat16, bits=None, device="mojo"):
        """Pages of zeros: of `dtype`, or of 4 bits with bits=4."""
        shape = (num_pages, kv_heads, page_size)
        if bits is None:
            return cls(*(torch.zeros(*shape, head_dim, dtype=dtype, device=device) for _ in range(2)))
        if bits != 4 or head_dim % GROUP:
            raise ValueError(f"PagedKVCache: bits must be 4 (or None), head_dim a multiple of {GROUP}; got {bits}, {head_dim}")
        codes = (torch.zeros(*shape, head_dim // 2, dtype=torch.uint8, device=device) for _ in range(2))
        scales = (torch.zeros(*shape, head_dim // GROUP, 2, dtype=torch.float16, device=device) for _ in range(2))
        return cls(*codes, *scales)


def _overlaps(t) -> bool:
    """Whether two elements of t may share memory."""
    extent = 1
    for size, stride in sorted(zip(t.shape, t.stride()), key=lambda x: x[1]):
        if size == 1:
            continue
        if stride < extent:
            return True
        extent += (size - 1) * stride
    return False


def _share(a, b) -> bool:
    """Whether two tensors with contiguous rows share memory; also where that
    takes too long to tell, which layouts of pages do not.

    A byte of both is a solution of sum n_s * s = the distance of their first
    bytes, give or take a row, with a term for each stride s: of a, of b
    negated, or of both.  From the largest on, a stride's multiples are tried
    that the smaller ones can make up for: one or two of them, in tensors
    whose dimensions lie inside one another."""
    at = [t._ptr if isinstance(t, TorchMojoTensor) else t.data_ptr() for t in (a, b)]
    rows = [t.shape[-1] * t.element_size() for t in (a, b)]
    terms = {}  # stride in bytes -> the least and the greatest n
    for t, sign in ((a, 1), (b, -1)):
        for size, stride in zip(t.shape[:-1], t.stride()):
            low, high = terms.get(stride * t.element_size(), (0, 0))
            n = sign * (size - 1)
            terms[stride * t.element_size()] = (low + min(n, 0), high + max(n, 0))
    terms = sorted(terms.items(), reverse=True)
    reach = [(1 - rows[1], rows[0] - 1)]  # of the row, then of the smaller strides as well
    for s, (low, high) in reversed(terms):
        reach.append((reach[-1][0] + low * s, reach[-1][1] + high * s))
    reach.reverse()
    tries = 0

    def solve(i, rest) -> bool:
        nonlocal tries
        tries += 1
        low, high = reach[i]
        if not low <= rest <= high or tries > 20000:
            return tries > 20000
        if i == len(terms):
            return True
        (s, (least, most)), (low, high) = terms[i], reach[i + 1]
        if s == 0:
            return solve(i + 1, rest)
        return any(solve(i + 1, rest - n * s) for n in range(max(least, -((high - rest) // s)), min(most, (rest - low) // s) + 1))

    return solve(0, at[1] - at[0])


# ---------------------------------------------------------------------------
# the plain formulas (off the mojo device)
# ---------------------------------------------------------------------------
def pack(x):
    """(codes uint8 [..., d / 2], scales float16 [..., d / 32, 2]) of x
    [..., d]: 32-bit word g * (d / 32) + s of a row holds channels
    32 s + 8 g + e, channel e in nibble e / 2 + 4 (e % 2)."""
    *lead, d = x.shape
    n = d // GROUP
    x = x.double().reshape(*lead, n, GROUP)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    x = x.clamp(-_LIMIT, _LIMIT)
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scales = torch.cat([(high - low) / 15.0, low], dim=-1).float().half()
    scales = torch.where(bad, torch.full_like(scales, float("nan")), scales)
    step, base = scales[..., :1].double(), scales[..., 1:].double()
    codes = torch.where(step > 0, ((x - base) / torch.where(step > 0, step, 1.0)).round().clamp(0, 15), 0.0)
    words = codes.to(torch.uint8).reshape(*lead, n, 4, 4, 2).transpose(-1, -2).transpose(-4, -3)
    words = words.reshape(*lead, d // 2, 2)
    return words[..., 0] | (words[..., 1] << 4), scales


def unpack(codes, scales):
    """The f32 values that codes and scales stand for."""
    *lead, half = codes.shape
    n = half // 16
    x = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(*lead, 4, n, 2, 4)
    x = x.transpose(-1, -2).transpose(-4, -3).reshape(*lead, n, GROUP).float()
    scales = scales.float()
    return (scales[..., 1:] + scales[..., :1] * x).flatten(-2)


def _places(cache, table, starts, tokens, counts, wanted=None):
    """(real, page, slot) [batch, tokens] of each token, or of the wanted ones."""
    t = torch.arange(tokens)
    pos = starts.long()[:, None] + t
    real = (t < counts[:, None]) if counts is not None else torch.ones_like(pos, dtype=torch.bool)
    if wanted is not None:
        real = wanted
    place = pos // cache.page_size
    bad = real & ((pos < 0) | (place >= table.shape[1]))
    if bad.any():
        raise IndexError("a position or page of a paged cache is out of range")
    place = torch.where(real, place, 0)
    page = table.long().gather(1, place) if table.shape[1] else place
    if (real & ((page < 0) | (page >= cache.num_pages))).any():
        raise IndexError("a position or page of a paged cache is out of range")
    return real, torch.where(real, page, 0), pos % cache.page_size


def append_plain(cache, table, starts, k, v, cos, sin, q, counts):
    real, page, slot = _places(cache, table, starts, k.shape[2], counts)
    out = None
    if cos is not None:
        pos = starts.long()[:, None] + torch.arange(k.shape[2])
        if (real & (pos >= cos.shape[0])).any():
            raise IndexError("a position or page of a paged cache is out of range")
        pos = torch.where(real, pos, 0)
        wide = torch.float64 if cache.bits == 4 else torch.float32
        c, s = cos[pos][:, None].to(wide), sin[pos][:, None].to(wide)

        def turn(x):
            half = x.shape[-1] // 2
            x = x.to(wide)
            return x * c + torch.cat([-x[..., half:], x[..., :half]], dim=-1) * s

        if q is not None:
            out = torch.where(real[:, None, :, None], turn(q), 0.0).to(q.dtype)
        k = turn(k)
    rows = (page[real], slice(None), slot[real])
    for pages, scales, x in ((cache.k, cache.k_scales, k), (cache.v, cache.v_scales, v)):
        x = x.transpose(1, 2)[real]
        if scales is None:
            pages[rows] = x.to(pages.dtype)
        else:
            pages[rows], scales[rows] = pack(x)
    return out


def gather_plain(cache, table, starts, length, counts, dtype, wanted=None):
    real, page, slot = _places(cache, table, starts, length, counts, wanted)

    def rows(pages, scales):
        x = pages[page, :, slot] if scales is None else unpack(pages[page, :, slot], scales[page, :, slot])
        return torch.where(real[:, :, None, None], x.to(dtype), 0.0).to(dtype).transpose(1, 2)

    return rows(cache.k, cache.k_scales), rows(cache.v, cache.v_scales)


def attention_plain(q, cache, table, starts, counts, window, sinks, scale):
    b, h, t, d = q.shape
    n = counts if counts is not None else torch.full((b,), t)
    n = n.clamp(0, t)
    ends = torch.where(n > 0, starts + n, 0)
    _places(cache, table, torch.where(n > 0, starts, 0), t, n)  # the queries' own places exist
    length = int(ends.max()) if b else 0
    i = torch.where(torch.arange(t) < n[:, None], starts[:, None] + torch.arange(t), -1)[:, None, :, None]
    j = torch.arange(length)
    keep = j <= i
    if window:
        keep = keep & ((i - j < window) | (j < sinks))
    wanted = keep.any(2)[:, 0]
    k, v = gather_plain(cache, table, torch.zeros_like(starts), length, ends, torch.float32, wanted)
    g = h // cache.kv_heads
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = (q.float() @ k.transpose(-1, -2) * scale).masked_fill(~keep, float("-inf"))
    p = torch.where(keep.any(-1, keepdim=True), torch.softmax(s, dim=-1), 0.0)
    return (p @ v).to(q.dtype)
