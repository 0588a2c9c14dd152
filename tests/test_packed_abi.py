"""Refusals of the entry points of packed sequences, rotary positions and token
log-probabilities: each is made on the host, before any launch (no GPU)."""

import ctypes

import pytest

from test_library import raw  # noqa: F401  (the fixture)

EINVAL, EUNSUPPORTED, EWORKSPACE = 1, 3, 4
P = 0x10000  # an aligned address that no call may use
F32, BF16, F16, I32, I64 = 0, 1, 2, 5, 4


@pytest.fixture
def lib(raw):  # noqa: F811
    from torch_mojo_backend.eager_kernels import SIGNATURES

    for name, (res, args) in SIGNATURES.items():
        if "packed" in name or "rope_at" in name or "logprobs" in name:
            getattr(raw, name).restype, getattr(raw, name).argtypes = res, args
    raw.mi355x_last_error.restype = ctypes.c_char_p
    return raw


def refused(lib, call, name, cases):
    for rc, over in cases:
        assert call(lib, **over) == rc, over
        assert lib.mi355x_last_error().startswith(name), over


def plan(lib, **over):
    a = dict(plan=P, bytes=1 << 20, positions=P, offsets=P, n=3, tokens=100, error=None, stream=None)
    assert not set(over) - set(a)
    return lib.mi355x_packed_plan(*{**a, **over}.values())


def test_plan(lib):
    refused(lib, plan, b"mi355x_packed_plan", [
        (EINVAL, dict(n=-1)), (EINVAL, dict(tokens=-1)), (EINVAL, dict(tokens=1 << 30)), (EINVAL, dict(n=1 << 30)),
        (EINVAL, dict(plan=None)), (EINVAL, dict(offsets=None)), (EINVAL, dict(positions=None)), (EINVAL, dict(plan=P + 8)),
        (EWORKSPACE, dict(bytes=64 + 16 * 10))])
    assert lib.mi355x_packed_plan_bytes(-1, 5) == -1 and lib.mi355x_packed_plan_bytes(3, 1 << 30) == -1
    # a tile of every full 128 and 64 rows, one more a sequence, and two of padding
    assert lib.mi355x_packed_plan_bytes(3, 1000) == 64 + 16 * ((7 + 3 + 2) + (15 + 3 + 2))


def th(*s):
    return (ctypes.c_int64 * 2)(*s)


ROWS = dict(tokens=100, heads=4, kv_heads=2, d=64, scale=0.1, window=0, dtype=BF16)
BAD = [(EINVAL, dict(tokens=-1)), (EINVAL, dict(tokens=1 << 30)), (EINVAL, dict(n=-1)), (EINVAL, dict(heads=0)),
       (EINVAL, dict(kv_heads=0)), (EINVAL, dict(heads=3)), (EINVAL, dict(heads=1 << 16, kv_heads=1)), (EINVAL, dict(window=-1)),
       (EINVAL, dict(scale=float("nan"))), (EINVAL, dict(scale=float("inf"))), (EINVAL, dict(scale=1e38)),
       (EUNSUPPORTED, dict(d=60)), (EUNSUPPORTED, dict(d=264)), (EUNSUPPORTED, dict(d=0)), (EUNSUPPORTED, dict(dtype=3)),
       (EINVAL, dict(tokens=1 << 28, heads=8)), (EINVAL, dict(lse=None)), (EINVAL, dict(plan=None)), (EINVAL, dict(plan=P + 4)),
       (EINVAL, dict(q=None)), (EINVAL, dict(k=P + 8)), (EINVAL, dict(vt=th(128, 60))), (EINVAL, dict(qt=th(-256, 64))),
       (EINVAL, dict(kt=th(1 << 26, 64))), (EINVAL, dict(low=P + 8))]


def forward(lib, **over):
    s = th(256, 64)
    a = dict(o=P, ot=s, low=None, lse=P, q=P, qt=s, k=P, kt=s, v=P, vt=s, plan=P, n=3, **ROWS, stream=None)
    assert not set(over) - set(a)
    return lib.mi355x_packed_attn_fwd(*{**a, **over}.values())


def backward(lib, **over):
    s = th(256, 64)
    a = dict(dq=P, dqt=s, dk=P, dkt=s, dv=P, dvt=s, do=P, dot=s, q=P, qt=s, k=P, kt=s, v=P, vt=s, o=P, ot=s, low=None, lse=P,
             plan=P, n=3, **ROWS, ws=P, wsb=1 << 30, stream=None)
    assert not set(over) - set(a)
    return lib.mi355x_packed_attn_bwd(*{**a, **over}.values())


def test_attention(lib):
    refused(lib, forward, b"mi355x_packed_attn_fwd", [*BAD, (EINVAL, dict(o=None)), (EINVAL, dict(ot=th(256, 63)))])
    refused(lib, backward, b"mi355x_packed_attn_bwd", [*BAD, (EINVAL, dict(dq=None)), (EINVAL, dict(do=P + 2)), (EINVAL, dict(o=None)),
                                                       (EINVAL, dict(dvt=th(250, 64))), (EWORKSPACE, dict(ws=None)),
                                                       (EWORKSPACE, dict(wsb=100))])
    assert forward(lib, tokens=0) == 0 and backward(lib, tokens=0) == 0
    for dtype in (BF16, F32):
        need = lib.mi355x_packed_attn_bwd_workspace_bytes(3, 100, 4, 2, 64)
        assert backward(lib, wsb=need - 1, dtype=dtype) == EWORKSPACE
    assert lib.mi355x_packed_attn_bwd_workspace_bytes(3, 100, 4, 4, 64) < need


def rope(lib, **over):
    s = (ctypes.c_int64 * 3)(1280, 64, 256)
    a = dict(qo=P, qot=s, q=P, qt=s, heads=4, ko=P, kot=s, k=P, kt=s, kv_heads=1, positions=P, pdt=I32, pst=0, freq=P, batch=2,
             seq=5, d=64, turned=64, laced=0, scale=1.0, inverse=0, dtype=BF16, stream=None)
    assert not set(over) - set(a)
    return lib.mi355x_rope_at(*{**a, **over}.values())


def test_rope(lib):
    refused(lib, rope, b"mi355x_rope_at", [
        (EINVAL, dict(batch=-1)), (EINVAL, dict(seq=-1)), (EINVAL, dict(heads=-1)), (EINVAL, dict(kv_heads=-1)), (EINVAL, dict(d=0)),
        (EINVAL, dict(turned=63)), (EINVAL, dict(turned=66)), (EINVAL, dict(turned=-2)), (EINVAL, dict(pdt=F32)),
        (EUNSUPPORTED, dict(d=4104)), (EINVAL, dict(heads=1 << 16)), (EINVAL, dict(seq=1 << 31)), (EINVAL, dict(scale=float("nan"))),
        (EINVAL, dict(scale=1e39)), (EINVAL, dict(q=None)), (EINVAL, dict(ko=None)), (EINVAL, dict(positions=None)),
        (EINVAL, dict(freq=None)), (EUNSUPPORTED, dict(dtype=3))])
    assert rope(lib, batch=0) == 0 and rope(lib, heads=0, kv_heads=0) == 0


def logprobs(lib, **over):
    a = dict(lp=P, ent=P, stats=P, tlp=P, tt=P, x=P, dtype=BF16, ld=50, tokens=P, n=3, c=50, top=5, ignore=-100, error=None, ws=P,
             wsb=1 << 30, stream=None)
    assert not set(over) - set(a)
    return lib.mi355x_token_logprobs_fwd(*{**a, **over}.values())


def gradient(lib, **over):
    a = dict(dx=P, ld_dx=56, x=P, dtype=BF16, ld=50, stats=P, ent=P, tokens=P, tt=P, top=5, dlp=P, dent=P, dtop=P, n=3, c=50,
             ignore=-100, stream=None)
    assert not set(over) - set(a)
    return lib.mi355x_token_logprobs_bwd(*{**a, **over}.values())


def test_logprobs(lib):
    both = [(EINVAL, dict(n=-1)), (EINVAL, dict(c=0)), (EINVAL, dict(c=1 << 31)), (EINVAL, dict(n=1 << 23)), (EINVAL, dict(ld=-1)),
            (EINVAL, dict(top=-1)), (EINVAL, dict(top=51)), (EUNSUPPORTED, dict(top=65, c=100)), (EUNSUPPORTED, dict(dtype=3)),
            (EINVAL, dict(x=None)), (EINVAL, dict(tokens=None)), (EINVAL, dict(tt=None))]
    refused(lib, logprobs, b"mi355x_token_logprobs_fwd", [*both, (EINVAL, dict(tlp=None)),
                                                          (EWORKSPACE, dict(c=262144, ws=None)), (EWORKSPACE, dict(c=262144, wsb=100))])
    refused(lib, gradient, b"mi355x_token_logprobs_bwd", [*both, (EINVAL, dict(dx=None)), (EINVAL, dict(stats=None)),
                                                          (EINVAL, dict(ent=None)), (EINVAL, dict(ld_dx=49))])
    assert logprobs(lib, n=0) == 0 and gradient(lib, n=0) == 0
    ws = lib.mi355x_token_logprobs_workspace_bytes
    assert ws(0, 50, 5, BF16) == 0 and ws(1000, 50257, 5, BF16) == 0
    assert ws(-1, 50, 5, BF16) == ws(1, 50, 65, BF16) == ws(1, 50, 5, I64) == -1
    need = ws(1, 262144, 20, BF16)
    assert need > 0 and logprobs(lib, n=1, c=262144, top=20, wsb=need - 1) == EWORKSPACE
