"""The paged cache's operations one after another on the MI355X: a model that
answers token by token, and the operations themselves over many calls."""

import pytest
import torch

import decode_cases as cases
from paged_cases import Case, check, np64
from torch_mojo_backend import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _mojo(mojo):
    return mojo


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("head_dim,window,page", [(64, 7, 4), (256, 40, 16)])
def test_calls_of_any_length_give_the_prefill(dtype, head_dim, window, page):
    m, ref = cases.model(dtype, "mojo", head_dim=head_dim, window=window)
    n = 120
    idx = cases.tokens(3, n)
    with torch.no_grad():
        want = ref(idx)
        whole = m(idx.to("mojo")).cpu().double()
    steps = [[70, 1, 33], [1, 1, 1], [4, 0, 4], [0, 64, 17], [1, 1, 1], [5, 5, 0]]
    steps.append([n - sum(s[i] for s in steps) for i in range(3)])
    lim = cases.bound(dtype, want, 4 * head_dim)
    assert (whole - want).abs().max() <= lim
    for s in (steps, [[1, 1, 1]] * n):
        got = cases.run(m, idx, s, "mojo", page=page)
        assert (got - want).abs().max() <= lim


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, None), (torch.float16, None), (torch.float32, None),
                                        (torch.bfloat16, 4), (torch.float32, 4)])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 24), (256, 16), (96, 8)])
def test_many_calls(dtype, bits, d, page):
    """Each call's attention against f64 over the rows that the cache reads back."""
    hk, h, b = 2, 4, 3
    c = Case([0] * b, page=page, bits=bits, device="mojo", d=d, hk=hk, dtype=dtype)
    width = -(-180 // page)
    cache = type(c.cache).zeros(b * width, page, hk, d, dtype=dtype, bits=bits)
    c.cache = cache
    c.table = torch.randperm(b * width, generator=torch.Generator().manual_seed(9)).view(b, width).int()
    c.dev_table = c.table.to("mojo")
    g = torch.Generator().manual_seed(8)
    ang = torch.rand(180, d // 2, generator=g).repeat(1, 2) * 6.2
    cos, sin = ang.cos().to("mojo"), ang.sin().to("mojo")
    at = [0] * b
    for counts in ([40, 17, 0], [1, 1, 1], [1, 0, 1], [33, 64, 2], [1, 1, 1], [5, 5, 5]):
        t = max(counts)
        q, k, v = (torch.randn(b, t, n, d, generator=g).to(dtype).to("mojo").transpose(1, 2) for n in (h, hk, hk))
        turned = ops.paged_append(cache, c.dev_table, c.ints(at), k, v, cos, sin, q=q, counts=c.ints(counts))
        ends = [a + n for a, n in zip(at, counts)]
        c.lengths = ends
        c.values = [np64(x) for x in ops.paged_gather(cache, c.dev_table, c.ints([0] * b), max(ends), counts=c.ints(ends))]
        for window, sinks in ((0, 0), (20, 3)):
            o = ops.paged_attention(turned, cache, c.dev_table, c.ints(at), counts=c.ints(counts), window=window, sinks=sinks)
            check(o, *c.expected(turned.cpu(), at, counts, window, sinks), f"{counts} window {window}")
        at = ends


@pytest.mark.parametrize("weights", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [None, 4])
def test_under_autocast(weights, bits):
    m, ref = cases.model(weights, "mojo", head_dim=64, window=7)
    idx = cases.tokens(3, 60)
    with torch.no_grad():
        want = ref(idx)
        with torch.autocast("mojo", dtype=torch.bfloat16):
            got = cases.run(m, idx, [[30, 1, 7], [1, 1, 1], [29, 58, 52]], "mojo", bits=bits)
    assert torch.isfinite(got).all()
    assert bits == 4 or (got - want).abs().max() <= cases.bound(torch.bfloat16, want, 4 * 64)
