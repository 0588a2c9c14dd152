"""Refusals of the paged cache's and the sinks' entry points of the library:
each is made on the host, before any launch (no GPU)."""

import ctypes

import pytest

from test_library import raw  # noqa: F401  (the fixture)

EINVAL, EUNSUPPORTED, EWORKSPACE = 1, 3, 4
P = 0x1000  # an aligned address that no call may use
F32, BF16, F16 = 0, 1, 2


def bht(*s):
    return (ctypes.c_int64 * 3)(*s)


@pytest.fixture
def lib(raw):  # noqa: F811
    from torch_mojo_backend.eager_kernels import SIGNATURES

    for name, (res, args) in SIGNATURES.items():
        if "paged" in name or "sink" in name:
            getattr(raw, name).restype, getattr(raw, name).argtypes = res, args
    raw.mi355x_last_error.restype = ctypes.c_char_p
    return raw


def cache(bits=0, d=64, dtype=BF16, pages=4, page=16, heads=2, **over):
    from torch_mojo_backend.eager_kernels import PagedCache

    c = PagedCache()
    width = d // 2 if bits == 4 else d
    c.k = c.v = P
    c.k_phs[:] = c.v_phs[:] = (heads * page * width, page * width, width)
    if bits == 4:
        n = d // 32 * 2
        c.k_scales = c.v_scales = P
        c.ks_phs[:] = c.vs_phs[:] = (heads * page * n, page * n, n)
    c.num_pages, c.page_size, c.kv_heads, c.d, c.dtype, c.bits = pages, page, heads, d, dtype, bits
    for name, value in over.items():
        if isinstance(value, tuple):
            getattr(c, name)[:] = value
        else:
            setattr(c, name, value)
    return c


def append(lib, c, **over):
    a = dict(table=P, stride=3, width=3, starts=P, counts=None, k=P, kb=bht(128, 64, 64), v=P, vb=bht(128, 64, 64), qo=None,
             qob=bht(0, 0, 0), q=None, qb=bht(0, 0, 0), cos=None, sin=None, rdt=0, rlen=0, batch=1, heads=0, seq=1,
             dtype=BF16, error=None, stream=None)
    assert not set(over) - set(a)
    return lib.mi355x_paged_append(c, *{**a, **over}.values())


def attend(lib, c, **over):
    a = dict(o=P, ob=bht(128, 64, 64), q=P, qb=bht(128, 64, 64), cache=c, table=P, stride=3, width=3, starts=P, counts=None,
             batch=1, heads=2, seq=1, scale=0.1, window=0, sinks=0, dtype=BF16, ws=None, wsb=0, error=None, stream=None)
    assert not set(over) - set(a)
    return lib.mi355x_paged_attn(*{**a, **over}.values())


def gather(lib, c, **over):
    a = dict(k=P, kb=bht(128, 64, 64), v=P, vb=bht(128, 64, 64), cache=c, table=P, stride=3, width=3, starts=P, counts=None,
             batch=1, seq=1, dtype=BF16, error=None, stream=None)
    assert not set(over) - set(a)
    return lib.mi355x_paged_gather(*{**a, **over}.values())


@pytest.mark.parametrize("call", [append, attend, gather])
def test_caches_that_are_refused(lib, call):
    bad = [(EUNSUPPORTED, dict(dtype=7)), (EINVAL, dict(bits=8)), (EUNSUPPORTED, dict(d=60)), (EUNSUPPORTED, dict(d=512)),
           (EUNSUPPORTED, dict(bits=4, d=48)), (EINVAL, dict(heads=0)), (EINVAL, dict(heads=1 << 16)), (EINVAL, dict(pages=0)),
           (EINVAL, dict(pages=1 << 31)), (EINVAL, dict(page=0)), (EINVAL, dict(k=None)), (EINVAL, dict(bits=4, v_scales=None)),
           (EINVAL, dict(k=P + 8)), (EINVAL, dict(v_phs=(2048, 1024, 60))), (EINVAL, dict(k_phs=(-2048, 1024, 64))),
           (EINVAL, dict(bits=4, ks_phs=(128, 65, 4))), (EINVAL, dict(bits=4, k_scales=P + 2))]
    for rc, over in bad:
        keep = {k: over[k] for k in ("bits", "d", "dtype", "pages", "page", "heads") if k in over}
        c = cache(**keep, **{k: v for k, v in over.items() if k not in keep})
        assert call(lib, c) == rc, over
        assert lib.mi355x_last_error().startswith(b"mi355x_paged")


@pytest.mark.parametrize("call", [append, attend, gather])
def test_sequences_that_are_refused(lib, call):
    bad = [dict(batch=-1), dict(batch=1 << 16), dict(seq=-1), dict(seq=1 << 31), dict(width=-1), dict(width=1 << 31),
           dict(starts=None), dict(table=None)]
    for over in bad:
        assert call(lib, cache(), **over) == EINVAL, over
    assert call(lib, cache(), dtype=7) == EUNSUPPORTED
    assert call(lib, cache(), batch=0) == 0 and call(lib, cache(), seq=0) == 0


def test_appends_that_are_refused(lib):
    for over in (dict(dtype=F32), dict(cos=P), dict(cos=P, sin=P, rdt=F16), dict(cos=P, sin=P, rlen=-1), dict(q=P, qo=P, heads=2),
                 dict(cos=P, sin=P, q=P, heads=2), dict(heads=2), dict(cos=P, sin=P, q=P, qo=P, heads=1 << 16), dict(k=None),
                 dict(k=P + 8), dict(vb=bht(128, 60, 64)), dict(cos=P + 4, sin=P),
                 dict(cos=P, sin=P, q=P, qo=P, heads=2, qb=bht(128, 64, 4))):
        assert append(lib, cache(), **over) == EINVAL, over
    assert append(lib, cache(d=24, k_phs=(768, 384, 24), v_phs=(768, 384, 24)), cos=P, sin=P) == EINVAL
    assert append(lib, cache(), batch=1 << 15, seq=1 << 16) == EINVAL


def test_attentions_that_are_refused(lib):
    for over in (dict(dtype=F32), dict(heads=3), dict(heads=0), dict(heads=1 << 16), dict(window=-1), dict(sinks=-1),
                 dict(scale=float("nan")), dict(o=None), dict(q=None), dict(q=P + 8), dict(qb=bht(128, 60, 64)),
                 dict(seq=1 << 30)):
        assert attend(lib, cache(), **over) == EINVAL, over
    assert attend(lib, cache(d=96, k_phs=(1536, 768, 96), v_phs=(1536, 768, 96)), batch=1 << 10, seq=1 << 13) == EINVAL
    long = dict(width=1000)
    need = lib.mi355x_paged_attn_workspace_bytes(cache(), 1000, 1, 2, 1, 0, 0, BF16)
    assert need > 0 and attend(lib, cache(), **long) == EWORKSPACE
    assert attend(lib, cache(), ws=P, wsb=need - 1, **long) == EWORKSPACE


def test_windows_that_are_refused(lib):
    s = bht(64 * 64, 64, 64)

    def fwd(**over):
        a = dict(o=P, os=s, low=None, lse=P, q=P, qs=s, k=P, ks=s, v=P, vs=s, batch=1, heads=2, hk=2, sq=64, skv=64, d=64, scale=0.1,
                 window=8, sinks=1, dtype=BF16, stream=None)
        assert not set(over) - set(a)
        return lib.mi355x_attn_fwd_sink(*{**a, **over}.values())

    def bwd(ws=None, **over):
        a = dict(dq=P, dqs=s, dk=P, dks=s, dv=P, dvs=s, do=P, dos=s, q=P, qs=s, k=P, ks=s, v=P, vs=s, o=P, os=s, low=None, lse=P, batch=1,
                 heads=2, hk=2, sq=64, skv=64, d=64, scale=0.1, window=8, sinks=1, dtype=BF16, ws=ws, wsb=0, stream=None)
        assert not set(over) - set(a)
        return lib.mi355x_attn_bwd_sink(*{**a, **over}.values())

    for call in (fwd, bwd):
        for over in (dict(window=0), dict(window=-1), dict(sinks=-1), dict(heads=3), dict(hk=0), dict(sq=0), dict(batch=0)):
            assert call(**over) == EINVAL, over
        assert call(dtype=7) == EUNSUPPORTED and call(d=257) == EUNSUPPORTED
    assert bwd() == EWORKSPACE and bwd(ws=P) == EWORKSPACE
    size = lib.mi355x_attn_bwd_sink_workspace_bytes
    # positions past the sequence change nothing
    assert size(1, 2, 2, 64, 64, 64, 1 << 62, 1 << 62) == size(1, 2, 2, 64, 64, 64, 64, 64) > 0


def test_workspaces_of_many_sinks(lib):
    """Nothing for sinks that hide nothing, and for others no multiple of what they are."""
    def size(b, h, hk, t, d, window, sinks):
        return lib.mi355x_attn_bwd_sink_workspace_bytes(b, h, hk, t, t, d, window, sinks)

    for b, h, hk, t, d, window, sinks in ((1, 12, 12, 8192, 64, 16, 8192), (1, 12, 12, 8192, 64, 16, 8176), (1, 4, 2, 500, 128, 400, 100)):
        assert size(b, h, hk, t, d, window, sinks) == size(b, h, hk, t, d, t, 0)
    assert size(1, 12, 12, 8192, 64, 16, 8175) > size(1, 12, 12, 8192, 64, 16, 0)
    for b, h, hk, t, d, window, sinks in ((1, 32, 32, 32768, 128, 512, 1024), (1, 12, 12, 32768, 64, 512, 4096), (1, 12, 12, 8192, 64, 16, 4000),
                                          (8, 16, 4, 32768, 64, 256, 65), (1, 4, 1, 4096, 256, 512, 4), (64, 64, 64, 100000, 64, 1, 64)):
        more = size(b, h, hk, t, d, window, sinks) - size(b, h, hk, t, d, window, 0)
        # 4096 blocks of 128 keys and each block's own, four times the last one's, dK and dV in f32
        assert 0 < more <= 2 * 4 * d * (4 * 4096 * 128 + 2 * b * h * sinks), (t, sinks)
    assert size(0, 2, 2, 64, 64, 8, 1) >= 0


@pytest.mark.parametrize("dtype,h,hk,t,d,sinks", [
    (F32, 64, 64, 131072, 64, 65536), (BF16, 64, 64, 131072, 64, 65536), (BF16, 32, 1, 2 ** 27, 64, 1),
    (BF16, 4096, 4096, 2 ** 18, 64, 0)])
def test_window_backwards_of_too_many_blocks(lib, dtype, h, hk, t, d, sinks):
    """Sums in 1024 threads, of sinks and of grouped heads, and blocks: refused before the first launch."""
    s = bht(t * d, d, d)
    assert lib.mi355x_attn_bwd_sink(P, s, P, s, P, s, P, s, P, s, P, s, P, s, P, s, None, P, 1, h, hk, t, t, d, 0.1, 1, sinks, dtype, P,
                                    1 << 62, None) == EINVAL
    assert b"blocks" in lib.mi355x_last_error() or b"sums" in lib.mi355x_last_error() or b"threads" in lib.mi355x_last_error()


def test_windows_past_every_position_share_keys_as_none(lib):
    size = lib.mi355x_paged_attn_workspace_bytes
    none = size(cache(), 1000, 1, 2, 1, 0, 0, BF16)
    for window, sinks in ((1 << 62, 1 << 62), ((1 << 63) - 1, 1), (1, (1 << 63) - 1), (1 << 20, 0)):
        assert size(cache(), 1000, 1, 2, 1, window, sinks, BF16) == none > 0
    assert size(cache(), 1000, 1, 2, 1, 100, 4, BF16) == 0


@pytest.mark.parametrize("kw,dtype,alone", [(dict(d=64), BF16, 384), (dict(d=128), F16, 384), (dict(d=256), BF16, 256), (dict(d=64, dtype=F32), F32, 384),
                                            (dict(d=128, dtype=F32), F32, 256), (dict(d=256, dtype=F32), F32, 128), (dict(d=96), BF16, 128),
                                            (dict(d=128, bits=4), BF16, 384), (dict(d=256, bits=4), F16, 256), (dict(d=128, bits=4), F32, 128)])
def test_keys_that_one_block_takes(lib, kw, dtype, alone):
    c = cache(heads=1, **kw)
    size = lambda keys, window=0: lib.mi355x_paged_attn_workspace_bytes(c, keys // 16, 1, 4, 1, window, 0, dtype)  # noqa: E731
    assert size(alone) == 0 and size(10 ** 5, alone) == 0
    assert size(alone + 16) > 0 and size(10 ** 5, alone + 1) > 0
    many = lambda keys: lib.mi355x_paged_attn_workspace_bytes(c, keys // 16, 200, 4, 1, 0, 0, dtype)  # noqa: E731
    assert many(384) == 0 and many(400) > 0
