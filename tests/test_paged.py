"""The paged cache off the GPU: the oracle, the plain formulas, the refusals,
and the mojo path's argument packing over the stand-in of the library."""

import copy

import numpy as np
import pytest
import torch

import paged_standin  # noqa: F401  (adds the cache's entry points to the stand-in)
from oracle import paged as oracle
from paged_cases import Case, check, np64
from torch_mojo_backend import ops
from torch_mojo_backend.kv_cache import PagedKVCache, pack, unpack


@pytest.fixture(params=["cpu", "mojo"])
def device(request, mojo):
    if request.param == "mojo" and mojo != "host":
        pytest.skip("the stand-in is for machines without a GPU")
    return request.param


# ---- the oracle ----
def test_oracle_places_fill_a_row():
    for d in (32, 64, 96, 256):
        got = sorted(oracle.place_of(c, d) for c in range(d))
        assert got == sorted((b, n) for b in range(d // 2) for n in range(2))


def test_oracle_quantize_is_within_half_a_step():
    x = np.random.default_rng(0).normal(size=(50, 64)) * 3
    codes, scale, low = oracle.quantize(x)
    err = np.abs(oracle.values(codes, scale, low) - x).reshape(50, 2, 32)
    # half a step, and what rounding the scale (15 of them) and the minimum to f16 moves
    assert (err <= scale.astype(float)[..., None] * (0.5 + 15 * 2.0 ** -11) + np.abs(low.astype(float))[..., None] * 2.0 ** -11).all()
    grid = np.arange(16.0).repeat(2) - 5
    codes, scale, low = oracle.quantize(grid)
    assert scale == [1.0] and low == [-5.0] and (oracle.values(codes, scale, low) == grid).all()


def test_oracle_attention_closed_forms():
    rng = np.random.default_rng(1)
    k, v = rng.normal(size=(2, 1, 9, 8))
    q = rng.normal(size=(2, 1, 8))
    assert np.allclose(oracle.attend(q, k, v, [0]), v[0, 0])          # one visible key
    assert np.allclose(oracle.attend(q, k, v, [5], window=1), v[0, 5])
    assert (oracle.attend(q, k, v, [-1]) == 0).all()
    assert np.allclose(oracle.attend(q, 0 * k, v, [8], window=3, sinks=2), v[0, [0, 1, 6, 7, 8]].mean(0))
    o, _ = oracle.window_forward(*rng.normal(size=(3, 1, 1, 9, 8)), 3, 2)
    assert o.shape == (1, 1, 9, 8)


def test_oracle_window_backward_is_the_difference_quotient():
    rng = np.random.default_rng(2)
    do, q = rng.normal(size=(2, 1, 4, 7, 8))
    k, v = rng.normal(size=(2, 1, 2, 7, 8))
    got = oracle.window_backward(do, q, k, v, 3, 1)
    loss = lambda: (oracle.window_forward(q, k, v, 3, 1)[0] * do).sum()  # noqa: E731
    for x, dx in zip((q, k, v), got):
        for i in [(0, 0, 0, 0), (0, 1, 2, 5), (0, 1, 6, 7), (0, 0, 4, 3)]:
            x[i] += 1e-5
            up = loss()
            x[i] -= 2e-5
            down = loss()
            x[i] += 1e-5
            assert abs((up - down) / 2e-5 - dx[i]) < 1e-8 + 1e-7 * abs(dx[i])


# ---- plain formulas and the mojo path over the stand-in ----
@pytest.mark.parametrize("d", [32, 64, 96, 256])
def test_pack_matches_the_oracle(d):
    x = torch.randn(5, 3, d, generator=torch.Generator().manual_seed(d)).bfloat16()
    x[0, 0, 3] = float("nan")
    x[1, 1, d - 1] = float("inf")
    x[2, 2] = 1.5
    x[3, 0, 0] = 1e6  # of f32 range
    codes, scales = pack(x)
    c, s, m = oracle.quantize(x.double().numpy())
    for ch in range(d):
        byte, nibble = oracle.place_of(ch, d)
        assert ((codes[..., byte].numpy() >> (4 * nibble) & 15) == c[..., ch]).all()
    assert np.array_equal(scales.numpy()[..., 0], s, equal_nan=True) and np.array_equal(scales.numpy()[..., 1], m, equal_nan=True)
    back = unpack(codes, scales).double().numpy()
    want = oracle.values(c, s, m)
    assert np.allclose(back, want, rtol=2.0 ** -23, atol=0, equal_nan=True)
    assert np.isnan(back[0, 0, :32]).all() and (back[2, 2] == 1.5).all()


@pytest.mark.parametrize("bits", [None, 4])
@pytest.mark.parametrize("page,slots_first", [(16, False), (24, True), (1, False)])
def test_append_then_gather(device, bits, page, slots_first):
    starts, counts = [0, 5, 17, 0], [3, 0, 7, 7]
    c = Case([s + 7 for s in starts], page=page, bits=bits, device=device, slots_first=slots_first, dtype=torch.float32)
    t, d = 7, c.d
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(4, t, c.hk, d, generator=g).transpose(1, 2) for _ in range(2))
    q = torch.randn(4, t, 6, d, generator=g).transpose(1, 2)
    ang = torch.rand(64, d // 2, generator=g).repeat(1, 2) * 6
    cos, sin = ang.cos(), ang.sin()
    before = [x.cpu().clone() for x in (c.cache.k, c.cache.v)]
    rot = ops.paged_append(c.cache, c.dev_table, c.ints(starts), k.to(device), v.to(device), cos.to(device),
                           sin.to(device), q=q.to(device), counts=c.ints(counts))
    gk, gv = ops.paged_gather(c.cache, c.dev_table, c.ints(starts), t, counts=c.ints(counts))
    owned = set()
    for b in range(4):
        n = counts[b]
        pos = np.arange(starts[b], starts[b] + n)
        owned |= {(int(c.table[b, p // page]), p % page) for p in pos}
        wq, wk = (oracle.turn(np64(x[b, :, :n]), cos[pos].numpy(), sin[pos].numpy()) for x in (q, k))
        wv = np64(v[b, :, :n])
        check(rot[b, :, :n], wq, np.full(wq.shape, 2.0 ** -22 * 8), "q")
        assert (np64(rot[b, :, n:]) == 0).all() and (np64(gk[b, :, n:]) == 0).all()
        if bits == 4:
            wk, wv = (oracle.values(*oracle.quantize(x)) for x in (wk, wv))
        check(gk[b, :, :n], wk, np.full(wk.shape, 2.0 ** -22 * 8), "k")
        check(gv[b, :, :n], wv, np.full(wv.shape, 2.0 ** -23 * 8), "v")
    for x, old in zip((c.cache.k, c.cache.v), before):  # other slots are as they were
        x = x.cpu()
        for p in range(c.cache.num_pages):
            for s in range(page):
                if (p, s) not in owned:
                    assert torch.equal(x[p, :, s].nan_to_num(7.0), old[p, :, s].nan_to_num(7.0))


@pytest.mark.parametrize("bits", [None, 4])
@pytest.mark.parametrize("window,sinks", [(0, 0), (5, 0), (5, 3), (1, 1)])
def test_attention_matches_the_oracle(device, bits, window, sinks):
    starts, counts = [0, 9, 30, 4, 0], [2, 3, 3, 0, 0]
    c = Case([s + n for s, n in zip(starts, counts)], page=8, bits=bits, device=device, dtype=torch.float32)
    q = c.queries(4, 3)
    out = ops.paged_attention(q.to(device), c.cache, c.dev_table, c.ints(starts), counts=c.ints(counts),
                              window=window, sinks=sinks)
    check(out, *c.expected(q, starts, counts, window, sinks))


def test_pages_that_no_query_sees_are_not_looked_up(device):
    """Between the sinks' pages and the window's, and behind the last token."""
    c = Case([60, 40], page=4, device=device, dtype=torch.float32)
    c.table[0, 1:9], c.table[1, 1:4], c.table[1, 10:] = -1, 10 ** 6, -7  # windows begin at 57 - 20 + 1 and 18
    q = c.queries(2, 3)
    out = ops.paged_attention(q.to(device), c.cache, c.table.to(device), c.ints([57, 37]), window=20, sinks=4)
    check(out, *c.expected(q, [57, 37], [3, 3], 20, 4))
    c.cache.k.cpu()


def test_lengths_of_zero_and_one(device):
    c = Case([1, 1], page=4, device=device, dtype=torch.float32)
    q = c.queries(2, 1)
    out = ops.paged_attention(q.to(device), c.cache, c.dev_table, c.ints([0, 0]))
    assert (np64(out) == np.stack([c.values[1][b][:, :1] for b in range(2)])).all()
    empty = torch.zeros(2, 2, 0, 64).to(device)
    assert ops.paged_append(c.cache, c.dev_table, c.ints([0, 0]), empty, empty) is None
    assert ops.paged_attention(empty, c.cache, c.dev_table, c.ints([0, 0])).shape == (2, 2, 0, 64)
    assert ops.paged_gather(c.cache, c.dev_table, c.ints([0, 0]), 0)[0].shape == (2, 2, 0, 64)


def test_positions_and_pages_out_of_range_raise(device):
    for starts, table in (([0, 7], None), ([-1, 0], None), ([0, 0], 99), ([0, 0], -1)):
        c = Case([4, 4], page=4, device=device, dtype=torch.float32)
        tab = c.dev_table if table is None else torch.full((2, 1), table, dtype=torch.int32).to(device)
        x = torch.zeros(2, 2, 1, 64).to(device)
        for call in (lambda: ops.paged_append(c.cache, tab, c.ints(starts), x, x),
                     lambda: ops.paged_gather(c.cache, tab, c.ints(starts), 1),
                     lambda: ops.paged_attention(x, c.cache, tab, c.ints(starts))):
            with pytest.raises(IndexError, match="paged cache"):
                call()
                c.cache.k.cpu()
    c = Case([4, 4], page=4, device=device, dtype=torch.float32)
    cos = torch.zeros(3, 64).to(device)
    with pytest.raises(IndexError, match="paged cache"):
        ops.paged_append(c.cache, c.dev_table, c.ints([0, 3]), x, x, cos, cos)
        c.cache.k.cpu()


def test_refusals(device):
    c = Case([4, 4], page=4, device=device, dtype=torch.float32)
    s = c.ints([0, 0])
    x = torch.zeros(2, 2, 1, 64).to(device)
    cos = torch.zeros(8, 64).to(device)
    bad = [
        (ValueError, lambda: ops.paged_append(c.cache, c.dev_table, s, x[0], x)),
        (ValueError, lambda: ops.paged_append(c.cache, c.dev_table, s, x, x[:, :, :, :32])),
        (ValueError, lambda: ops.paged_append(c.cache, c.dev_table, s, x, torch.cat([x, x], 2))),
        (TypeError, lambda: ops.paged_append(c.cache, c.dev_table, s, x.bfloat16(), x.bfloat16())),
        (ValueError, lambda: ops.paged_append(c.cache, c.dev_table.long(), s, x, x)),
        (ValueError, lambda: ops.paged_append(c.cache, c.dev_table, s[:1], x, x)),
        (ValueError, lambda: ops.paged_append(c.cache, c.dev_table, s, x, x, cos)),
        (ValueError, lambda: ops.paged_append(c.cache, c.dev_table, s, x, x, cos[:, :32], cos[:, :32])),
        (TypeError, lambda: ops.paged_append(c.cache, c.dev_table, s, x, x, cos.double(), cos.double())),
        (ValueError, lambda: ops.paged_append(c.cache, c.dev_table, s, x, x, q=x)),
        (ValueError, lambda: ops.paged_append(c.cache, c.dev_table, s, x, x, cos, cos, q=x[:1])),
        (ValueError, lambda: ops.paged_attention(x[0], c.cache, c.dev_table, s)),
        (ValueError, lambda: ops.paged_attention(x[:, :1], c.cache, c.dev_table, s)),
        (TypeError, lambda: ops.paged_attention(x.half(), c.cache, c.dev_table, s)),
        (ValueError, lambda: ops.paged_attention(x, c.cache, c.dev_table, s, window=-1)),
        (ValueError, lambda: ops.paged_attention(x, c.cache, c.dev_table, s, window=3, sinks=-1)),
        (ValueError, lambda: ops.paged_attention(x, c.cache, c.dev_table, s, scale=float("inf"))),
        (ValueError, lambda: ops.paged_attention(x, c.cache, c.dev_table, s, counts=c.ints([1]))),
        (ValueError, lambda: ops.paged_gather(c.cache, c.dev_table, s, -1)),
        (TypeError, lambda: ops.paged_gather(c.cache, c.dev_table, s, 1, dtype=torch.int32)),
        (NotImplementedError, lambda: ops.paged_attention(x.clone().requires_grad_(), c.cache, c.dev_table, s)),
        (ValueError, lambda: PagedKVCache(x, x[:1])),
        (ValueError, lambda: PagedKVCache(x.expand(2, 2, 1, 64)[:, :1].expand(2, 2, 1, 64), x)),
        (ValueError, lambda: PagedKVCache(x[..., :20], x[..., :20])),
        (ValueError, lambda: PagedKVCache(x, x)),
        (ValueError, lambda: PagedKVCache(x, x[:])),
        (TypeError, lambda: PagedKVCache(x.int(), x.int())),
        (ValueError, lambda: PagedKVCache.zeros(2, 4, 1, 64, bits=8, device=device)),
        (ValueError, lambda: PagedKVCache.zeros(2, 4, 1, 48, bits=4, device=device)),
        (ValueError, lambda: PagedKVCache.zeros(2, 4, 1, 512, device=device)),
    ]
    if device == "mojo":
        bad.append((ValueError, lambda: ops.paged_attention(x.cpu(), c.cache, c.dev_table, s)))
        bad.append((ValueError, lambda: ops.paged_append(c.cache, c.dev_table.cpu(), s, x, x)))
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            raise AssertionError(f"call {i} was not refused")


def test_append_counts_as_a_write(device):
    c = PagedKVCache.zeros(2, 4, 1, 64, dtype=torch.float32, device=device)
    x = torch.ones(1, 1, 1, 64).to(device)
    before = c.k._version
    ops.paged_append(c, torch.zeros(1, 1, dtype=torch.int32).to(device), torch.zeros(1, dtype=torch.int32).to(device), x, x)
    assert c.k._version > before and float(c.k.cpu()[0, 0, 0].sum()) == 64


def test_no_sequences(device):
    c = Case([1], page=4, device=device, dtype=torch.float32)
    table, none = torch.zeros(0, 3, dtype=torch.int32).to(device), c.ints([])
    x = torch.zeros(0, 2, 5, 64).to(device)
    assert ops.paged_append(c.cache, table, none, x, x) is None
    assert ops.paged_attention(x, c.cache, table, none).shape == (0, 2, 5, 64)
    assert ops.paged_gather(c.cache, table, none, 3)[1].shape == (0, 2, 3, 64)


@pytest.mark.parametrize("bits", [None, 4])
def test_a_copy_of_a_cache_is_its_own(device, bits):
    c = PagedKVCache.zeros(2, 4, 1, 64, dtype=torch.float32, bits=bits, device=device)
    other = type(c)(*(t.clone() for t in c.tensors)) if device == "mojo" else copy.deepcopy(c)
    assert copy.copy(c).k is c.k
    x = torch.ones(1, 1, 1, 64).to(device)
    zero = torch.zeros(1, dtype=torch.int32).to(device)
    ops.paged_append(other, zero.view(1, 1), zero, x, x)
    assert (ops.paged_gather(c, zero.view(1, 1), zero, 1)[0].cpu() == 0).all()
    assert (ops.paged_gather(other, zero.view(1, 1), zero, 1)[0].cpu() == 1).all()


@pytest.mark.parametrize("far", [12, 500, 2 ** 30, 2 ** 31 - 2])
def test_positions_past_the_table_raise(device, far):
    c = Case([12, 12], page=4, device=device, dtype=torch.float32)
    x = torch.zeros(2, 2, 1, 64).to(device)
    for call in (lambda: ops.paged_append(c.cache, c.dev_table, c.ints([0, far]), x, x),
                 lambda: ops.paged_gather(c.cache, c.dev_table, c.ints([0, far]), 1),
                 lambda: ops.paged_attention(x, c.cache, c.dev_table, c.ints([0, far])),
                 lambda: ops.paged_attention(x, c.cache, c.dev_table, c.ints([0, far]), window=3, sinks=2)):
        with pytest.raises(IndexError, match="paged cache"):
            call()
            c.cache.k.cpu()


def test_pages_that_share_memory_are_refused(device):
    base = torch.zeros(9, 2, 4, 64).to(device)
    both = torch.zeros(8, 2, 2, 4, 64).to(device)
    codes = torch.zeros(4, 2, 8, 32, dtype=torch.uint8).to(device)
    scales = torch.zeros(5, 2, 8, 2, 2, dtype=torch.float16).to(device)
    other = torch.zeros(4, 2, 8, 2, 2, dtype=torch.float16).to(device)
    for k, v in ((base, base), (base[:2], base[1:3]), (base[:8], base[1:]), (base[:4, :1], base[3:7, :1]),
                 (base[:, :, :3], base[:, :, 1:]), (base[..., :32], base[..., 16:48]), (base[::2][:4], base[2::2])):
        with pytest.raises(ValueError, match="share memory"):
            PagedKVCache(k, v)
    with pytest.raises(ValueError, match="share memory"):
        PagedKVCache(codes, codes.clone(), scales[1:], scales[:4])
    for k, v in ((base[:4], base[4:8]), (base[::2][:4], base[1::2]), (base[:, :1], base[:, 1:]), (base[:, :, :2], base[:, :, 2:]),
                 (base[..., :32], base[..., 32:]), (both[:, 0], both[:, 1]), (both[:, :, 0], both[:, :, 1])):
        PagedKVCache(k, v)
    PagedKVCache(codes, codes.clone(), scales[:4], other)


def test_sharing_is_told_as_it_is():
    from torch_mojo_backend.kv_cache import _share

    g = np.random.default_rng(0)
    found = [0, 0]
    for _ in range(2000):
        flat = torch.zeros(4000, dtype=torch.uint8)

        def view():
            width, shape = int(g.integers(1, 9)), [int(n) for n in g.integers(1, 5, size=3)]
            strides = [int(g.choice([width + int(g.integers(0, 5)), 12, 40, 100, 130, 300])) for _ in range(3)]
            return flat.as_strided((*shape, width), (*strides, 1), int(g.integers(0, 200)))

        a, b = view(), view()
        places = [{int(i) for i in np.lib.stride_tricks.as_strided(np.arange(4000), x.shape, [8 * s for s in x.stride()])
                   .ravel() + x.storage_offset()} for x in (a, b)]
        want = bool(places[0] & places[1])
        assert _share(a, b) == _share(b, a) == want
        found[want] += 1
    assert min(found) > 200


@pytest.mark.parametrize("what", ["k", "v", "q", "none"])
def test_rows_of_the_pages_themselves(device, monkeypatch, what):
    """Tokens moved within the cache: the rows are read before any is written."""
    if device == "mojo":
        from host_standin import HostStandIn

        call, seen = HostStandIn.mi355x_paged_append, []

        def watched(self, cache, table, tst, width, starts, counts, *rest):
            seen.append([r.value if hasattr(r, "value") else r for r in (rest[0], rest[2], rest[6])])
            return call(self, cache, table, tst, width, starts, counts, *rest)

        monkeypatch.setattr(HostStandIn, "mi355x_paged_append", watched)
    n = 8
    c = PagedKVCache(*(torch.randn(1, 2, n, 64, generator=torch.Generator().manual_seed(i)).to(device) for i in range(2)))
    old = [x.cpu().clone() for x in (c.k, c.v)]
    rows = {x: torch.ones(1, 2, n - 1, 64).to(device) for x in "kvq"}
    if what != "none":
        rows[what] = (c.v if what == "v" else c.k)[:, :, :-1]
    cos, sin = torch.ones(n, 64).to(device), torch.zeros(n, 64).to(device)
    zero = torch.zeros(1, 1, dtype=torch.int32).to(device)
    out = ops.paged_append(c, zero, zero.view(1) + 1, rows["k"], rows["v"], cos, sin, q=rows["q"])
    for name, x, was in (("k", c.k, old[0]), ("v", c.v, old[1])):
        want = was[:, :, :-1] if what == name else torch.ones(1, 2, n - 1, 64)
        assert torch.equal(x.cpu()[:, :, 1:], want) and torch.equal(x.cpu()[:, :, :1], was[:, :, :1])
    assert torch.equal(out.cpu(), old[0][:, :, :-1] if what == "q" else torch.ones(1, 2, n - 1, 64))
    if device == "mojo":
        pages = [(t.data_ptr() if not hasattr(t, "_ptr") else t._ptr) for t in (c.k, c.v)]
        for ptr in seen[0]:
            assert not any(p <= ptr < p + 4 * 2 * n * 64 for p in pages)


@pytest.mark.parametrize("bits", [None, 4])
def test_a_caches_tensors_are_fixed(device, bits):
    """The kernels would go on using the old ones."""
    c = PagedKVCache.zeros(2, 4, 1, 64, dtype=torch.float32, bits=bits, device=device)
    for name in ("k", "v", "k_scales", "v_scales"):
        old = getattr(c, name)
        with pytest.raises(AttributeError, match="fixed"):
            setattr(c, name, old)
        assert getattr(c, name) is old
    c.note = 1  # other attributes are the user's
