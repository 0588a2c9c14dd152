"""Rows of packed attention, rotary positions and token log-probabilities that
lie past 2^31 elements of their tensors, on the MI355X against f64."""

import pytest
import torch

import logprob_cases
import packed_cases
import test_gpu_logprobs_long as long
from abi import CODE, call, i64, lib, p
from paged_cases import check

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _mojo(mojo):
    return mojo


def th(x):
    return i64(*x.stride()[:2])


@pytest.mark.parametrize("dtype,h,hk,d", [(BF, 32, 8, 128), (F32, 32, 8, 128), (BF, 16, 16, 256)])
def test_sequences_behind_many_rows(dtype, h, hk, d):
    """Two sequences at the end of a batch whose other rows, NaN, belong to none."""
    lengths, t = [200, 100], 2 ** 31 // (h * d) + 1000
    at, x = packed_cases.inputs(lengths, h, hk, d, dtype)
    first = t - 300
    rows = []
    for y in x:
        wide = torch.full((t, *y.shape[1:]), float("nan"), dtype=dtype, device="cuda")
        wide[first:] = y.cuda()
        rows.append(wide)
    q, k, v, dy = rows
    assert q.numel() > 2 ** 31
    out, dq, dk, dv = (torch.full_like(y, 7) for y in (q, q, k, v))
    low = torch.empty_like(q) if dtype is BF else None
    lse = torch.empty(h, t, device="cuda")
    n = len(lengths)
    offsets = torch.tensor([first + a for a in at], dtype=torch.int32, device="cuda")
    plan = torch.empty(lib().mi355x_packed_plan_bytes(n, t), dtype=torch.uint8, device="cuda")
    pos, error = torch.empty(t, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = torch.empty(lib().mi355x_packed_attn_bwd_workspace_bytes_for(n, t, h, hk, d, CODE[dtype]), dtype=torch.uint8, device="cuda")
    call("mi355x_packed_plan", p(plan), plan.numel(), p(pos), p(offsets), n, t, p(error), None)
    call("mi355x_packed_attn_fwd", p(out), th(out), p(low), p(lse), p(q), th(q), p(k), th(k), p(v), th(v), p(plan), n, t, h, hk, d,
         d ** -0.5, 0, CODE[dtype], None)
    call("mi355x_packed_attn_bwd", p(dq), th(dq), p(dk), th(dk), p(dv), th(dv), p(dy), th(dy), p(q), th(q), p(k), th(k), p(v), th(v),
         p(out), th(out), p(low), p(lse), p(plan), n, t, h, hk, d, d ** -0.5, 0, CODE[dtype], p(ws), ws.numel(), None)
    torch.cuda.synchronize()
    assert not error.item() and not pos[:first].any() and pos[first:].tolist() == [*range(200), *range(100)]
    want = packed_cases.expected(at, *x)
    for name, y in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        check(y[first:], *want[name], name)
        assert all(not part.any() for part in y[:first].split(1 << 16)), name


def test_tokens_behind_many_rows():
    h, d = 32, 128
    t = 2 ** 31 // (h * d) + 1000
    x = torch.randn(1, 100, h, d, generator=torch.Generator().manual_seed(0)).to(BF).transpose(1, 2)
    q = torch.zeros(t, h, d, dtype=BF, device="cuda")
    q[t - 100:] = x[0].transpose(0, 1).cuda()
    out = torch.empty_like(q)
    pos = torch.arange(t, dtype=torch.int32, device="cuda")
    f = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    bht, fm = i64(0, d, h * d), f.cuda()
    call("mi355x_rope_at", p(out), bht, p(q), bht, h, None, bht, None, bht, 0, p(pos), CODE[torch.int32], 0, p(fm), 1, t, d, d, 0, 1.0, 0,
         CODE[BF], None)
    torch.cuda.synchronize()
    want = logprob_cases.turned(x, torch.arange(t - 100, t), f, False, 1.0)
    check(out[t - 100:].transpose(0, 1)[None], *want)
    assert all(not part.any() for part in out[:t - 100].split(1 << 16))


@pytest.mark.parametrize("top", [0, 3])
def test_logits_behind_many_rows(top):
    c = 262144
    n = 2 ** 31 // c + 20
    gen = torch.Generator().manual_seed(1)
    x = (3.0 * torch.randn(4, c, generator=gen)).to(BF)
    tokens = torch.randint(0, c, (4,), generator=gen)
    g, gh = torch.randn(4, generator=gen), torch.randn(4, generator=gen)
    wide = torch.zeros(n, c, dtype=BF, device="cuda")
    wide[n - 4:] = x.cuda()
    dev = lambda *s, dt=F32: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    tk, gp, ge = dev(n, dt=torch.int64), dev(n), dev(n)
    for y, z in ((tk, tokens), (gp, g), (ge, gh)):
        y[n - 4:] = z.cuda()
    lp, ent, stats, tlp, tt, error = dev(n), dev(n), dev(n, 2), dev(n, 3), dev(n, 3, dt=torch.int64), dev(1, dt=torch.int32)
    dx = torch.empty_like(wide)
    ws = dev(max(16, lib().mi355x_token_logprobs_workspace_bytes(n, c, top, CODE[BF])), dt=torch.uint8)
    call("mi355x_token_logprobs_fwd", p(lp), p(ent), p(stats), p(tlp), p(tt), p(wide), CODE[BF], c, p(tk), n, c, top, -100, p(error), p(ws),
         ws.numel(), None)
    call("mi355x_token_logprobs_bwd", p(dx), c, p(wide), CODE[BF], c, p(stats), p(ent), p(tk), None, 0, p(gp), p(ge), None, n, c, -100, None)
    torch.cuda.synchronize()
    want = long.expected(x, tokens, g, gh)
    for name, y in (("logprobs", lp), ("entropy", ent), ("dx", dx)):
        check(y[n - 4:], *want[name], name)
    if top:
        assert tt[n - 4:].cpu().numpy().tolist() == logprob_cases.best_of(x, top).tolist()
        assert tt[:n - 4].unique().tolist() == [0, 1, 2]  # equal ones by index
    assert not error.item() and not dx[:n - 4].any()
