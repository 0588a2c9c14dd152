"""Token log-probabilities, entropy and top entries on the MI355X against f64."""

import numpy as np
import pytest
import torch

import logprob_cases as cases
from paged_cases import check
from torch_mojo_backend import ops

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _mojo(mojo):
    return mojo


def compare(got, want):
    for name in ("logprobs", "entropy", "top_logprobs"):
        value = getattr(got, name)
        if value is not None:
            value, (expected, bound) = value.detach().cpu().double(), want[name]
            hidden = np.isneginf(expected)  # (no difference can be taken there)
            assert np.array_equal(torch.isneginf(value).numpy(), hidden), name
            check(value.masked_fill(torch.from_numpy(hidden), 0.0), np.where(hidden, 0.0, expected), bound, name)
    if got.top_tokens is not None:
        assert np.array_equal(got.top_tokens.cpu().numpy(), want["top_tokens"])


def run(x, tokens, top=0, entropy=True, ignore_index=-100):
    got = ops.token_logprobs(x.to("mojo"), tokens.to("mojo"), top=top, entropy=entropy, ignore_index=ignore_index)
    compare(got, cases.expected(x, tokens, top, ignore_index=ignore_index))


def train(x, tokens, top=0, entropy=True, picked=True):
    n = x.shape[0]
    g = torch.Generator().manual_seed(7)
    grads = [torch.randn(n, generator=g) if picked else None, torch.randn(n, generator=g) if entropy else None,
             torch.randn(n, top, generator=g) if top else None]
    leaf = x.to("mojo").requires_grad_()
    got = ops.token_logprobs(leaf, tokens.to("mojo"), top=top, entropy=entropy)
    want = cases.expected(x, tokens, top, grads)
    compare(got, want)
    ends = [(y, g) for y, g in zip((got.logprobs, got.entropy, got.top_logprobs), grads) if g is not None]
    torch.autograd.backward([y for y, _ in ends], [g.to("mojo") for _, g in ends])
    check(leaf.grad, *want["dx"], "dx")


SIZES = [(1, 1, 1), (3, 7, 7), (2, 64, 5), (1, 1000, 64), (5, 2049, 5), (700, 2047, 3), (600, 8192, 20), (1, 8193, 1),
         (300, 50257, 5), (4, 50257, 20), (1, 262144, 20), (2, 262143, 64), (1, 200003, 0), (257, 65536, 2), (258, 65544, 2)]


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("n,c,top", SIZES)
def test_forward(dtype, n, c, top):
    run(*cases.logits(n, c, dtype), top)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("n,c,top,entropy,picked", [(1, 1, 1, True, True), (3, 9, 4, True, True), (600, 300, 0, False, True),
                                                    (70, 4099, 5, True, False), (5, 50257, 0, True, True),
                                                    (600, 50257, 1, True, True), (1, 262144, 20, True, True),
                                                    (513, 1000, 64, False, True)])
def test_gradients(dtype, n, c, top, entropy, picked):
    train(*cases.logits(n, c, dtype), top, entropy, picked)


@pytest.mark.parametrize("dtype,top", [(BF, 0), (BF, 3), (F32, 0)])
def test_a_gradient_larger_than_the_cache(dtype, top):
    """A row's gradient is the same in a batch whose gradient has over 256 MB."""
    n, times, c = 600, 5, 50257
    x, tokens = cases.logits(n, c, dtype)

    def grad(x, tokens):
        leaf = x.to("mojo").requires_grad_()
        got = ops.token_logprobs(leaf, tokens.to("mojo"), top=top, entropy=True)
        weight = torch.linspace(-1, 1, n).repeat(len(tokens) // n).to("mojo")
        loss = (got.logprobs * weight).sum() + (got.entropy * weight).sum()
        if top:
            loss = loss + (got.top_logprobs * weight[:, None]).sum()
        loss.backward()
        return leaf.grad.cpu()

    want, got = grad(x, tokens), grad(x.repeat(times, 1), tokens.repeat(times))
    for part in got.chunk(times):
        assert torch.equal(part, want)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,c", [(2, 50), (600, 3000), (3, 50257), (300, 50257)])
def test_ties(dtype, n, c):
    """All equal, two values, steps of a few values, and 0 with -0."""
    for x in (torch.zeros(n, c), torch.randint(0, 2, (n, c)).float(), torch.randint(0, 9, (n, c)).float(),
              torch.where(torch.arange(c) % 3 == 0, -0.0, 0.0).expand(n, c)):
        run(x.to(dtype), torch.randint(0, c, (n,)), 33)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,c", [(4, 40), (600, 2000), (4, 50257), (300, 50257)])
def test_masked_vocabulary(dtype, n, c):
    """Entries of -inf: none but one left, half of them, the type's lowest value."""
    x, tokens = cases.logits(n, c, dtype)
    half = x.clone()
    half[:, ::2] = -torch.inf
    one = torch.full_like(x, -torch.inf)
    one[:, 5] = 3.0
    low = x.clone()
    low[:, ::2] = torch.finfo(dtype).min
    for y in (half, one, low):
        best = torch.from_numpy(cases.best_of(y, 20))
        run(y, best[:, 0], 5 if y is half else 20)
        train(y, best[:, 0], 1)
    got = ops.token_logprobs(half.to("mojo"), torch.full((n,), 4).to("mojo")).logprobs
    assert torch.isneginf(got.cpu()).all()


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("n,c,entropy", [(600, 9001, True), (600, 9001, False), (8, 50257, True), (8, 50257, False)])
def test_far_and_masked_rows_without_top_entries(dtype, n, c, entropy):
    """What a row's walk meets late, early or everywhere: large values, -inf, the type's lowest."""
    x, tokens = cases.logits(n, c, dtype)
    low = torch.finfo(dtype).min
    x[0, :], x[0, c - 2] = -torch.inf, 3.0
    x[1, :] = low
    x[2, 1::2] = low
    x[3, c // 2] = 40000.0
    x[4, :] = -40000.0
    x[5, :c // 2], x[5, c // 2:] = -30000.0, 30000.0
    x[6, c - 1] = 60000.0
    x[7, :4000] = -torch.inf
    tokens[:8] = torch.tensor([c - 2, 7, 8, c // 2, c - 1, c - 1, c - 1, 4000])
    run(x, tokens, 0, entropy)
    train(x, tokens, 0, entropy)


@pytest.mark.parametrize("n,c", [(3, 100), (600, 1000), (2, 50257), (300, 50257)])
def test_nan_and_infinity(n, c):
    """A NaN makes its row NaN and comes first; so do a +inf, and a row of -inf."""
    x, tokens = cases.logits(n, c, F32)
    x[0, 17] = float("nan")
    x[0, 3] = float("nan")
    x[1, 9] = float("inf")
    x[2:3] = float("-inf")
    got = ops.token_logprobs(x.to("mojo"), tokens.to("mojo"), top=4, entropy=True)
    bad = min(n, 3)
    for y in (got.logprobs, got.entropy, got.top_logprobs):
        assert torch.isnan(y.cpu()[:bad]).all()
        assert not torch.isnan(y.cpu()[bad:]).any()
    order = got.top_tokens.cpu()
    assert order[0, :2].tolist() == [3, 17] and order[1, 0] == 9
    if n > 2:
        assert order[2].tolist() == [0, 1, 2, 3]
    assert np.array_equal(order[bad:].numpy(), cases.best_of(x[bad:], 4) if n > bad else np.zeros((0, 4)))


def test_ignored_and_bad_tokens():
    x, tokens = cases.logits(6, 500, BF)
    tokens[1] = tokens[4] = -100
    run(x, tokens)
    train(x, tokens)
    tokens[1] = tokens[4] = 7
    run(x, tokens, ignore_index=7)
    for bad in (-1, 500, 2 ** 40):
        tokens[2] = bad
        got = ops.token_logprobs(x.to("mojo"), tokens.to("mojo")).logprobs
        with pytest.raises(IndexError):
            got.cpu()
        assert got.cpu()[2] == 0


def test_shapes_and_strides():
    x, tokens = cases.logits(6, 501, BF)
    want = cases.expected(x, tokens, 4)
    wide = torch.zeros(6, 508, dtype=BF)
    wide[:, 3:504] = x
    for y in (wide.to("mojo")[:, 3:504], x.t().contiguous().to("mojo").t()):
        compare(ops.token_logprobs(y, tokens.to("mojo"), top=4, entropy=True), want)
    got = ops.token_logprobs(x.view(2, 3, 501).to("mojo"), tokens.view(2, 3).to("mojo"), top=4, entropy=True)
    assert got.top_tokens.shape == (2, 3, 4) and got.logprobs.shape == (2, 3)
    compare(type(got)(*(y.view(6, *y.shape[2:]) for y in got)), want)
    got = ops.token_logprobs(x[0].to("mojo"), tokens[0].to("mojo"), top=4, entropy=True)
    assert got.logprobs.shape == () and got.top_logprobs.shape == (4,)
    one = ops.token_logprobs(x[:1].to("mojo").expand(5, 501), tokens[:5].to("mojo"))
    check(one.logprobs, *cases.expected(x[:1].expand(5, 501), tokens[:5])["logprobs"])
    none = ops.token_logprobs(x[:0].to("mojo"), tokens[:0].to("mojo"), top=2, entropy=True)
    assert none.top_logprobs.shape == (0, 2) and none.entropy.shape == (0,)
    assert ops.token_logprobs(x.to("mojo"), top=3).logprobs is None
    leaf = x.view(2, 3, 501).to("mojo").requires_grad_()
    ops.token_logprobs(leaf, tokens.view(2, 3).to("mojo")).logprobs.sum().backward()
    check(leaf.grad.view(6, 501), *cases.expected(x, tokens, 0, (torch.ones(6), None, None))["dx"])


def test_far_from_zero():
    """Logits with a large common part, which must cost nothing but their own steps."""
    x, tokens = cases.logits(5, 3001, F32)
    run(x + 4096.0, tokens, 3)
    run(x * 30, tokens, 3)


def test_no_second_gradient():
    x, tokens = cases.logits(2, 30, F32)
    leaf = x.to("mojo").requires_grad_()
    dx, = torch.autograd.grad(ops.token_logprobs(leaf, tokens.to("mojo")).logprobs.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="second time"):
        dx.sum().backward()
