"""The paged cache on the MI355X against f64: appending, reading back and
attention, over types, head layouts, page sizes, lengths and masks."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import paged as oracle
from paged_cases import STEP, Case, check, np64
from torch_mojo_backend import ops
from torch_mojo_backend.kv_cache import PagedKVCache

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _mojo(mojo):
    return mojo


def _tables(n, d, dtype, seed=4):
    ang = torch.rand(n, d // 2, generator=torch.Generator().manual_seed(seed)).repeat(1, 2) * 6.2
    return ang.cos().to(dtype), ang.sin().to(dtype)


@pytest.mark.parametrize("dtype,bits,d,page,rope", [
    (BF, None, 256, 16, F32), (BF, None, 64, 24, BF), (HF, None, 128, 8, F32), (F32, None, 80, 1, F32),
    (BF, 4, 128, 64, F32), (HF, 4, 64, 24, HF), (F32, 4, 96, 16, F32), (BF, 4, 32, 3, BF), (BF, 4, 256, 16, None),
    (BF, None, 24, 16, None)])
def test_append_then_gather(dtype, bits, d, page, rope):
    starts, counts = [0, 5, 1000, 0, 63], [37, 0, 21, 37, 1]
    t, hk, h = 37, 3, 6
    c = Case([s + t for s in starts], page=page, bits=bits, device="mojo", d=d, hk=hk, dtype=dtype, slots_first=page == 8)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(5, t, hk, d, generator=g).to(dtype).transpose(1, 2) for _ in range(2))
    q = torch.randn(5, t, h, d, generator=g).to(dtype).transpose(1, 2)
    cos, sin = _tables(1100, d, rope) if rope else (None, None)
    before = [x.cpu().clone() for x in (c.cache.k, c.cache.v)]
    up = lambda x: x.to("mojo") if x is not None else None  # noqa: E731
    rot = ops.paged_append(c.cache, c.dev_table, c.ints(starts), up(k), up(v), up(cos), up(sin),
                           q=up(q) if rope else None, counts=c.ints(counts))
    out = F32 if bits == 4 else dtype
    gk, gv = ops.paged_gather(c.cache, c.dev_table, c.ints(starts), t, counts=c.ints(counts))
    owned = set()
    for b in range(5):
        n = counts[b]
        pos = np.arange(starts[b], starts[b] + n)
        owned |= {(int(c.table[b, p // page]), p % page) for p in pos}
        wq, wk, wv = (np64(x[b, :, :n]) for x in (q, k, v))
        if rope:
            wq, wk = (oracle.turn(x, np64(cos)[pos], np64(sin)[pos]) for x in (wq, wk))
            # a sum of two products in f32, each at most 6 (N(0, 1) rows), rounded once
            check(rot[b, :, :n], wq, STEP[dtype] * np.abs(wq) + 12 * 2.0 ** -23, "q")
            assert (np64(rot[b, :, n:]) == 0).all()
        assert (np64(gk[b, :, n:]) == 0).all() and (np64(gv[b, :, n:]) == 0).all()
        if bits == 4 and n:
            # the codes are those of the f64 rows; values leave in f32
            wk, wv = (oracle.values(*oracle.quantize(x)) for x in (wk, wv))
            check(gk[b, :, :n], wk, 2.0 ** -23 * 6 + 0 * wk, "k")
            check(gv[b, :, :n], wv, 2.0 ** -23 * 6 + 0 * wv, "v")
        elif n:
            check(gk[b, :, :n], wk, STEP[out] * np.abs(wk) + (12 * 2.0 ** -23 if rope else 0), "k")
            assert (np64(gv[b, :, :n]) == wv).all()
    for x, old in zip((c.cache.k, c.cache.v), before):
        x = x.cpu()
        for p in range(c.cache.num_pages):
            for s in range(page):
                if (p, s) not in owned:
                    assert torch.equal(x[p, :, s].nan_to_num(7.0), old[p, :, s].nan_to_num(7.0)), (p, s)


def test_scales_round_by_way_of_f32():
    """(max - min) / 15 just above the middle of two f16 values, nearer to it
    than f32 resolves: the f32 value is the middle, which goes to the even one."""
    x = torch.zeros(1, 1, 2, 32)
    x[..., 1] = -1.0
    x[..., 0] = torch.tensor([float.fromhex("0x1.d247fep-1"), float.fromhex("0x1.d8d802p-1")])
    _, scale, low = oracle.quantize(x.double().numpy())
    direct = ((x[..., 0].double().numpy() + 1.0) / 15.0).astype(np.float16)
    assert (direct != scale[..., 0]).all()  # the inputs tell the two apart
    c = PagedKVCache.zeros(1, 2, 1, 32, bits=4)
    zero = torch.zeros(1, 1, dtype=torch.int32).to("mojo")
    ops.paged_append(c, zero, zero.view(1), x.to("mojo"), x.to("mojo"))
    for scales in (c.k_scales, c.v_scales):
        got = scales.cpu().numpy()[0, 0, :, 0]
        assert (got[:, 0] == scale[0, 0, :, 0]).all() and (got[:, 1] == low[0, 0, :, 0]).all()


def _attention(c, h, starts, counts, t, dtype=None, window=0, sinks=0, scale=None):
    q = c.queries(h, t, dtype)
    strided = q.transpose(1, 2).contiguous().to("mojo").transpose(1, 2)
    out = ops.paged_attention(strided, c.cache, c.dev_table, c.ints(starts), counts=c.ints(counts), window=window,
                              sinks=sinks, scale=scale)
    check(out, *c.expected(q, starts, counts, window, sinks, scale), f"T{t} window {window} sinks {sinks}")


@pytest.mark.parametrize("dtype,bits", [(BF, None), (HF, None), (F32, None), (BF, 4), (HF, 4), (F32, 4)])
@pytest.mark.parametrize("d,hk,h", [(64, 3, 3), (128, 2, 8), (256, 1, 4), (96, 2, 2), (32, 1, 5)])
@pytest.mark.parametrize("page", [16, 24, 1])
def test_attention_of_one_token(dtype, bits, d, hk, h, page):
    starts = [0, 1, 16, 31, 32, 33, 200, 517, 0]
    counts = [1] * 8 + [0]
    c = Case([s + n for s, n in zip(starts, counts)], page=page, bits=bits, device="mojo", d=d, hk=hk, dtype=dtype)
    _attention(c, h, starts, counts, 1, dtype)
    _attention(c, h, starts, counts, 1, dtype, window=33, sinks=5, scale=0.3)


@pytest.mark.parametrize("dtype,bits", [(BF, None), (HF, None), (F32, None), (BF, 4)])
@pytest.mark.parametrize("d,hk,h,t", [(64, 2, 2, 5), (128, 2, 8, 4), (256, 1, 4, 9), (128, 1, 16, 3), (64, 1, 1, 70),
                                      (256, 1, 2, 33), (96, 1, 3, 6)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (16, 0), (40, 70), (1, 1)])
def test_attention_of_several_tokens(dtype, bits, d, hk, h, t, window, sinks):
    starts, counts = [0, 3, 90, 250, 0], [t, 1, t, max(t - 2, 1), 0]
    c = Case([s + n for s, n in zip(starts, counts)], page=16, bits=bits, device="mojo", d=d, hk=hk, dtype=dtype)
    _attention(c, h, starts, counts, t, dtype, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype,bits", [(BF, None), (F32, None), (BF, 4)])
@pytest.mark.parametrize("d", [64, 256])
def test_attention_over_a_long_sequence(dtype, bits, d):
    c = Case([9001, 130], page=64, bits=bits, device="mojo", d=d, hk=1, dtype=dtype)
    _attention(c, 4, [9000, 129], [1, 1], 1, dtype)
    _attention(c, 4, [9000, 129], [1, 1], 1, dtype, window=4096, sinks=100)


@pytest.mark.parametrize("dtype,bits", [(BF, None), (F32, None), (BF, 4), (HF, 4)])
@pytest.mark.parametrize("d,hk,h,page", [(64, 1, 4, 16), (128, 2, 4, 24), (256, 1, 2, 64), (80, 1, 2, 16)])
def test_attention_of_a_prompt(dtype, bits, d, hk, h, page):
    d = 96 if bits and d == 80 else d  # 4-bit rows are multiples of 32 channels
    c = Case([700, 431], page=page, bits=bits, device="mojo", d=d, hk=hk, dtype=dtype)
    _attention(c, h, [100, 0], [600, 431], 600, dtype)
    _attention(c, h, [100, 0], [600, 431], 600, dtype, window=64, sinks=20)


@pytest.mark.parametrize("d,h", [(64, 2), (128, 4), (256, 4), (64, 20), (128, 20)])
@pytest.mark.parametrize("page", [16, 24])
def test_f16_queries_over_4_bits_round_nothing_but_the_result(d, h, page):
    c = Case([700, 90], page=page, bits=4, device="mojo", d=d, hk=1, dtype=HF)
    c.bits = None  # the bound without a row's and a weight's rounding to f16
    _attention(c, h, [697, 88], [3, 2], 3, HF)
    _attention(c, h, [699, 89], [1, 1], 1, HF, window=100, sinks=3)


@pytest.mark.parametrize("scale", [0.0, -0.4])
def test_scale_of_any_sign(scale):
    c = Case([77], device="mojo", d=128)
    _attention(c, 2, [70], [7], 7, BF, scale=scale)


def test_large_scores_do_not_overflow():
    for bits in (None, 4):
        c = Case([300], device="mojo", d=64, hk=1, dtype=HF if bits is None else BF, bits=bits, spread=40.0)
        _attention(c, 4, [299], [1], 1, HF if bits is None else BF, scale=1.0)


def test_hidden_numbers_stay_hidden():
    """NaN and infinities in keys and values that a query does not see."""
    for bits in (None, 4):
        c = Case([100], device="mojo", d=64, hk=1, bits=bits)
        bad = torch.full((1, 1, 40, 64), float("nan"), dtype=BF)
        bad[..., ::2] = float("inf")
        # positions 4 .. 43: neither sinks nor in the window of the queries at 96 .. 99
        ops.paged_append(c.cache, c.dev_table, c.ints([4]), bad.to("mojo"), bad.to("mojo"))
        for x in c.values:
            x[:, :, 4:44] = 0.0
        _attention(c, 2, [96], [4], 4, BF, window=20, sinks=4)
        _attention(c, 2, [99], [1], 1, BF, window=56, sinks=4)


@pytest.mark.parametrize("dtype,bits", [(BF, None), (F32, None), (BF, 4)])
@pytest.mark.parametrize("d,page", [(64, 16), (64, 4), (256, 48), (96, 16)])
def test_pages_that_no_query_sees_are_not_looked_up(dtype, bits, d, page):
    c = Case([600, 400], page=page, bits=bits, device="mojo", d=d, hk=1, dtype=dtype)
    # windows begin at 597 - 100 + 1 and 397 - 100 + 1, sinks end at 7
    c.table[0, -(-7 // page):498 // page], c.table[1, -(-7 // page):298 // page], c.table[1, -(-400 // page):] = -1, 10 ** 6, -7
    q = c.queries(2, 3, dtype)
    out = ops.paged_attention(q.to("mojo"), c.cache, c.table.to("mojo"), c.ints([597, 397]), window=100, sinks=7)
    check(out, *c.expected(q, [597, 397], [3, 3], 100, 7))  # reads the flag as well


def test_offsets_past_32_bits():
    pages, page, hk, d = 70_000, 16, 8, 256  # 2.3e9 values a tensor
    k, v = (torch.empty(pages, hk, page, d, dtype=BF, device="mojo") for _ in range(2))
    cache = PagedKVCache(k, v)
    last = torch.arange(pages - 4, pages, dtype=torch.int32).view(1, 4)
    g = torch.Generator().manual_seed(5)
    rows = [torch.randn(1, hk, 50, d, generator=g).to(BF) for _ in range(2)]
    zero = torch.zeros(1, dtype=torch.int32).to("mojo")
    ops.paged_append(cache, last.to("mojo"), zero, *(x.to("mojo") for x in rows))
    got = ops.paged_gather(cache, last.to("mojo"), zero, 50)
    for a, b in zip(got, rows):
        assert torch.equal(a.cpu(), b)
    q = torch.randn(1, 16, 1, d, generator=g).to(BF)
    out = ops.paged_attention(q.to("mojo"), cache, last.to("mojo"), zero + 49)
    want = oracle.attend(np64(q)[0], np64(rows[0])[0], np64(rows[1])[0], [49])
    check(out, want[None], STEP[BF] * np.abs(want[None]) + 1e-4)


def test_pages_out_of_range_are_left_out():
    c = Case([40], device="mojo", d=64, hk=1)
    x = torch.ones(1, 1, 1, 64, dtype=BF).to("mojo")
    for table in ([[0, 99, 1]], [[0, -5, 1]], [[0, 2 ** 31 - 1, 1]]):
        tab = torch.tensor(table, dtype=torch.int32).to("mojo")
        for call in (lambda: ops.paged_append(c.cache, tab, c.ints([20]), x, x),
                     lambda: ops.paged_gather(c.cache, tab, c.ints([20]), 3),
                     lambda: ops.paged_attention(x, c.cache, tab, c.ints([40]))):
            call()
            with pytest.raises(IndexError, match="paged cache"):
                x.cpu()
    x.cpu()  # the flag is cleared


@pytest.mark.parametrize("dtype,bits,d,n", [(BF, None, 64, 1), (F32, None, 128, 40), (HF, 4, 256, 1), (BF, None, 96, 1),
                                            (BF, 4, 64, 700), (BF, None, 96, 700)])
def test_visible_nan_is_seen(dtype, bits, d, n):
    """A sequence whose keys are NaN answers NaN, and its neighbour does not."""
    c = Case([n, n], page=16, bits=bits, device="mojo", d=d, hk=1, dtype=dtype)
    nan = torch.full((1, 1, n, d), float("nan"), dtype=dtype).to("mojo")
    tab = c.dev_table[:1]
    _, v = ops.paged_gather(c.cache, tab, c.ints([0]), n, dtype=dtype)
    ops.paged_append(c.cache, tab, c.ints([0]), nan, v)
    q = c.queries(2, 1, dtype)
    out = ops.paged_attention(q.to("mojo"), c.cache, c.dev_table, c.ints([n - 1, n - 1])).cpu()
    assert torch.isnan(out[0]).all()
    want, bound = c.expected(q, [0, n - 1], [0, 1])
    check(out[1:], want[1:], bound[1:])


def test_windows_past_every_position():
    c = Case([77], device="mojo", d=64)
    q = c.queries(4, 2)
    want = c.expected(q, [75], [2])
    for window, sinks in ((2 ** 31, 0), (2 ** 70, 2 ** 70), (3, 2 ** 40)):
        check(ops.paged_attention(q.to("mojo"), c.cache, c.dev_table, c.ints([75]), window=window, sinks=sinks), *want)


def test_shared_pages_and_repeated_results():
    """Sequences with a common prefix read the same pages; a call repeated gives the same bits."""
    c = Case([64, 64], page=16, device="mojo", d=128, hk=2)
    tab = c.table.clone()
    tab[1, :2] = tab[0, :2]
    for x in c.values:
        x[1][:, :32] = x[0][:, :32]
    q = c.queries(4, 1)
    args = (q.to("mojo"), c.cache, tab.to("mojo"), c.ints([63, 60]))
    first = ops.paged_attention(*args)
    check(first, *c.expected(q, [63, 60], [1, 1]))
    assert all(torch.equal(first.cpu(), ops.paged_attention(*args).cpu()) for _ in range(3))


def test_captured_and_replayed(kernels):
    """Append and attention captured into a graph through the C entry points;
    each replay reads the positions of the moment."""
    from torch_mojo_backend.eager_kernels import PagedCache, check as ok

    d, hk, h, page, n = 128, 2, 8, 16, 64
    g = torch.Generator().manual_seed(6)
    dev = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()  # noqa: E731
    kp, vp = torch.zeros(n, hk, page, d, dtype=BF, device="cuda"), torch.zeros(n, hk, page, d, dtype=BF, device="cuda")
    desc = PagedCache()
    desc.k, desc.v = kp.data_ptr(), vp.data_ptr()
    desc.k_phs[:] = desc.v_phs[:] = kp.stride()[:3]
    desc.num_pages, desc.page_size, desc.kv_heads, desc.d, desc.dtype = n, page, hk, d, 1
    table = torch.randperm(n, generator=g).int().view(1, n).cuda()
    starts = torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v, q = dev(1, hk, 1, d), dev(1, hk, 1, d), dev(1, h, 1, d)
    o = torch.empty_like(q)
    ws = kernels.mi355x_paged_attn_workspace_bytes(desc, n, 1, h, 1, 0, 0, 1)
    hold = torch.empty(max(ws, 1), dtype=torch.uint8, device="cuda")
    bht = lambda x: (ctypes.c_int64 * 3)(*x.stride()[:3])  # noqa: E731

    def step(stream):
        ok("append", kernels.mi355x_paged_append(
            desc, table.data_ptr(), n, n, starts.data_ptr(), None, k.data_ptr(), bht(k), v.data_ptr(), bht(v),
            None, None, None, None, None, None, 0, 0, 1, 0, 1, 1, None, stream))
        ok("attention", kernels.mi355x_paged_attn(
            o.data_ptr(), bht(o), q.data_ptr(), bht(q), desc, table.data_ptr(), n, n, starts.data_ptr(), None,
            1, h, 1, d ** -0.5, 0, 0, 1, hold.data_ptr(), ws, None, stream))

    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step(side.cuda_stream)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            step(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    ks, vs = [], []
    for i in range(40):
        k.copy_(dev(1, hk, 1, d)), v.copy_(dev(1, hk, 1, d)), q.copy_(dev(1, h, 1, d))
        starts.fill_(i)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ks.append(np64(k)[0, :, 0]), vs.append(np64(v)[0, :, 0])
        want = oracle.attend(np64(q)[0], np.stack(ks, 1), np.stack(vs, 1), [i])
        check(o, want[None], STEP[BF] * np.abs(want[None]) + 1e-4, f"replay {i}")


@pytest.mark.parametrize("dtype,bits,d,page", [(BF, None, 64, 16), (F32, None, 128, 24), (HF, 4, 256, 16), (BF, None, 96, 16),
                                               (F32, 4, 64, 5)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (9, 3)])
def test_positions_past_the_table_see_what_it_holds(dtype, bits, d, page, window, sinks):
    """A query behind the table's last place: an error at the next read, the
    table's keys alone, and no more work than they take."""
    n = 3 * page
    c = Case([n, n], page=page, bits=bits, device="mojo", d=d, hk=1, dtype=dtype)
    q = c.queries(4, 2, dtype)
    for far in (n - 1, n, 40 * n, 2 ** 30, 2 ** 31 - 300):
        out = ops.paged_attention(q.to("mojo"), c.cache, c.dev_table, c.ints([far, n - 2]), window=window, sinks=sinks)
        with pytest.raises(IndexError, match="paged cache"):
            out.cpu()
        want, bound = c.expected(q, [far, n - 2], [0, 2], window, sinks)
        k, v = (x[0] for x in c.values)
        for t in range(2):  # the query sees j <= far + t < ..., of which the table has n
            j = np.arange(n)
            keep = (j <= far + t) & ((far + t - j < window) | (j < sinks) if window else True)
            if keep.any():
                s = d ** -0.5 * np64(q)[0, :, t] @ k[0, keep].T
                p = np.exp(s - s.max(-1, keepdims=True))
                want[0, :, t] = p / p.sum(-1, keepdims=True) @ v[0, keep]
        # the bound of the sequence beside it, of as many keys and the same spread, twice
        bound[0] = 2 * bound[1].max() + STEP[dtype] * np.abs(want[0])
        check(out, want, bound, f"position {far}")
    c.cache.k.cpu()  # the flag is cleared


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("d,turned", [(64, False), (64, True), (32, False), (96, True)])
def test_codes_are_of_clamped_values(dtype, d, turned):
    """Values on both sides of +-61440: the codes, too, are those of the clamped ones."""
    big = {F32: 70000.0, BF: 69632.0, HF: 65504.0}[dtype]
    low = {F32: 61425.0, BF: 61440.0, HF: 61408.0}[dtype]
    rows = torch.full((1, 1, 8, d), low)
    rows[..., 1::2] = big                    # the minimum's f16 is the limit
    rows[0, 0, 1] = -rows[0, 0, 1]
    rows[0, 0, 2, ::3] = -big                # both ends past it
    rows[0, 0, 3, 5:] = 0.0
    rows[0, 0, 4] = big
    rows[0, 0, 5] = torch.linspace(-2 * big, 2 * big, d)
    if dtype is F32:
        rows[0, 0, 6, 4:] = 3e38
    rows = rows.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max).to(dtype)
    cos, sin = torch.ones(8, d), torch.zeros(8, d)  # turned by nothing: the values in f64
    c = PagedKVCache.zeros(1, 8, 1, d, bits=4)
    zero = torch.zeros(1, 1, dtype=torch.int32).to("mojo")
    args = (cos.to("mojo"), sin.to("mojo")) if turned else ()
    ops.paged_append(c, zero, zero.view(1), rows.to("mojo"), rows.to("mojo"), *args)
    codes, scale, base = oracle.quantize(np64(rows))
    want = oracle.values(codes, scale, base)
    assert np.abs(want).max() <= 61440 + 16 + 15 * 2  # half a step of the minimum, and 15 of the scale
    for got in ops.paged_gather(c, zero, zero.view(1), 8):
        assert (np64(got) == want.astype(np.float32)).all()


@pytest.mark.parametrize("dtype,d", [(BF, 64), (F32, 96)])
def test_tokens_moved_within_the_pages(dtype, d):
    """Rows that are views of the pages are read before any is written."""
    n, hk = 4096, 3
    g = torch.Generator().manual_seed(7)
    old = [torch.randn(1, hk, n, d, generator=g).to(dtype) for _ in range(2)]
    c = PagedKVCache(*(x.to("mojo") for x in old))
    zero = torch.zeros(1, 1, dtype=torch.int32).to("mojo")
    ops.paged_append(c, zero, zero.view(1) + 1, c.k[:, :, :-1], c.v[:, :, :-1])
    for x, was in zip((c.k.cpu(), c.v.cpu()), old):
        assert torch.equal(x[:, :, 1:], was[:, :, :-1]) and torch.equal(x[:, :, :1], was[:, :, :1])


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("d,h", [(64, 1), (128, 20), (256, 4)])
def test_4_bit_values_at_the_ends_of_the_range(dtype, d, h):
    c = Case([90, 33], page=16, bits=4, device="mojo", d=d, hk=1, dtype=dtype)
    g = torch.Generator().manual_seed(9)
    v = ((torch.rand(2, 1, 90, d, generator=g) - 0.5) * 1e6).to(F32).to("mojo")  # most are clamped
    k, _ = ops.paged_gather(c.cache, c.dev_table, c.ints([0, 0]), 90, counts=c.ints([90, 33]))
    ops.paged_append(c.cache, c.dev_table, c.ints([0, 0]), k, v, counts=c.ints([90, 33]))
    c.values = [np64(x) for x in ops.paged_gather(c.cache, c.dev_table, c.ints([0, 0]), 90, counts=c.ints([90, 33]))]
    assert np.abs(c.values[1]).max() == 61440
    _attention(c, h, [89, 32], [1, 1], 1, dtype)
    _attention(c, h, [86, 29], [4, 4], 4, dtype, window=30, sinks=2)
