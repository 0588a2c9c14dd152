"""Appending to a paged cache and attending over it, as a model does it token
by token, off the GPU."""

import pytest
import torch

import decode_cases as cases
import paged_standin  # noqa: F401
from torch_mojo_backend.kv_cache import PagedKVCache


@pytest.fixture(params=["cpu", "mojo"])
def device(request, mojo):
    if request.param == "mojo" and mojo != "host":
        pytest.skip("the stand-in is for machines without a GPU")
    return request.param


STEPS = [[11, 4], [1, 1], [3, 2], [0, 5], [1, 1], [4, 7]]


def test_calls_of_any_length_give_the_prefill(device):
    m, ref = cases.model(torch.float32, device)
    idx = cases.tokens(2, 20)
    with torch.no_grad():
        want = ref(idx)
        whole = m(idx.to(device)).cpu().double()
    for steps in (STEPS, [[1, 1]] * 20, [[20, 20]]):
        got = cases.run(m, idx, steps, device)
        lim = cases.bound(torch.float32, want, 97)
        assert (got - want).abs().max() <= lim and (whole - want).abs().max() <= lim


def test_sinks_are_seen_by_local_layers_alone(device):
    m, _ = cases.model(torch.float32, device, sinks=0)
    s, _ = cases.model(torch.float32, device, sinks=2)
    idx = cases.tokens(1, 12)
    a, b = (cases.run(x, idx, [[12]], device) for x in (m, s))
    assert torch.equal(a[:, :7], b[:, :7]) and not torch.equal(a[:, 7:], b[:, 7:])


def test_pages_of_4_bits(device):
    m, _ = cases.model(torch.float32, device)
    idx = cases.tokens(2, 20)
    got = cases.run(m, idx, STEPS, device, bits=4)
    assert torch.isfinite(got).all()


def test_one_cache_a_layer(device):
    m, _ = cases.model(torch.float32, device)
    table = torch.zeros(1, 1, dtype=torch.int32).to(device)
    with pytest.raises(ValueError):
        m.forward_cached(torch.zeros(1, 1, dtype=torch.int64).to(device), m.caches(1, 4)[:2], table, table.view(1))


@pytest.mark.parametrize("weights", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("pages", [None, torch.float32, torch.bfloat16, 4])
def test_under_autocast(device, weights, pages):
    """Rows leave the projections in autocast's type; pages keep their own."""
    m, ref = cases.model(weights, device)
    if pages is not None:
        kw = {"bits": 4} if pages == 4 else {"dtype": pages}
        m.caches = lambda n, size, *, bits=None: [
            PagedKVCache.zeros(n, size, m.cfg.kv_heads, m.cfg.head_dim, device=device, **kw) for _ in m.blocks]
    idx = cases.tokens(2, 20)
    with torch.no_grad():
        want = ref(idx)
        with torch.autocast(device, dtype=torch.bfloat16):
            whole = m(idx.to(device)).cpu().double()
            got = cases.run(m, idx, STEPS, device)
        plain = cases.run(m, idx, STEPS, device)
    lim = cases.bound(torch.bfloat16, want, 97)
    assert (whole - want).abs().max() <= lim
    for x in (got, plain):
        assert torch.isfinite(x).all()
        assert pages == 4 or (x - want).abs().max() <= lim
