"""float16 attention's gradients where an operand of their products would leave
float16's range: gradients far below and far above 1, probabilities far below 1.

The gradients are linear in do, and a power of two takes every fp32 step along
exactly, so for f a power of two the gradients of f do are f times those of do,
rounded to float16: the bound of attention_64 for do, times f, and half a step of
float16's below its normal range."""
import math

import pytest
import torch

from token_helpers import STEP, attention_64

pytestmark = pytest.mark.gpu
T = torch.float16


def _rand(shape, seed, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * size).to(T)


def _grads(q, k, v, do, **how):
    from blitzgs_amd.attention import attention
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    return torch.autograd.grad(attention(*leaves, **how), leaves, do)


def _within(got, want, bound, what):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: {int((~torch.isfinite(got)).sum())} not finite"
    over = ((got - want).abs() / bound).max().item()
    assert over <= 1.0, f"{what}: {over:.3g} times the bound"


def _check(q, k, v, do, f, causal=False, key_lengths=None, scale=None):
    """The gradients of f do, f a power of two that makes do's elements no subnormals."""
    small = (do.double() * f).to(T)
    assert torch.equal(small.double(), do.double() * f)
    want = attention_64(q, k, v, causal, key_lengths, None, 1 / math.sqrt(q.shape[3]) if scale is None else scale, do)
    got = _grads(q, k, v, small, causal=causal, key_lengths=key_lengths, scale=scale)
    for name, g in zip(("dq", "dk", "dv"), got):
        value, bound = want[name]
        assert (value.abs() * f).max() < 6e4, "the true gradient fits"
        _within(g, f * value, f * bound + STEP[T], name)


def _away_from_zero(do, least):
    return torch.where(do.abs() < least, torch.full_like(do, least), do)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [64, 128, 33])
@pytest.mark.parametrize("f", [2.0 ** -10, 2.0 ** -13])
def test_small_gradients_over_thousands_of_keys(gpu, f, D, causal):
    Tq, Tk = 70, 3001
    q, k, v = _rand((1, 2, Tq, D), 1), _rand((1, 1, Tk, D), 2), _rand((1, 1, Tk, D), 3)
    do = _away_from_zero(_rand((1, 2, Tq, D), 4), 0.6)
    _check(q, k, v, do, f, causal)


@pytest.mark.parametrize("D", [64, 128, 33])
def test_small_gradients_of_many_queries(gpu, D):
    # dk's sums run over thousands of queries
    Tq, Tk = 3001, 70
    q, k, v = _rand((1, 2, Tq, D), 1), _rand((1, 2, Tk, D), 2), _rand((1, 2, Tk, D), 3)
    _check(q, k, v, _away_from_zero(_rand((1, 2, Tq, D), 4), 0.6), 2.0 ** -13)


@pytest.mark.parametrize("D", [64, 128, 40])
def test_large_gradients(gpu, D):
    # dS itself passes 65504; small keys and queries keep the true gradients below it
    Tq, Tk = 70, 64
    q, k = _rand((1, 2, Tq, D), 1, 2.0 ** -7), _rand((1, 2, Tk, D), 2, 2.0 ** -7)
    v, do = _rand((1, 2, Tk, D), 3, 8.0), _rand((1, 2, Tq, D), 4)
    v[:, :, 3] = 60.0
    do[:, :, 7] = 1.0 + do[:, :, 7].abs()
    _check(q, k, v, do.clamp(-3.5, 3.5), 2.0 ** 13, scale=1.0)


@pytest.mark.parametrize("which", ["early", "late"])
@pytest.mark.parametrize("by", ["key", "query"])
def test_one_sum_over_many_magnitudes(gpu, which, by):
    # values, and gradients, that grow or fall by 2^24 along the walk; the bound of
    # each result is its own sum's, in which the large ones lead
    Tq, Tk, D = 520, 520, 64
    q, k, v = _rand((1, 1, Tq, D), 1), _rand((1, 1, Tk, D), 2), _rand((1, 1, Tk, D), 3)
    do = _away_from_zero(_rand((1, 1, Tq, D), 4), 0.6)
    along = torch.arange(520, device="cuda") * 24 // 520 - 12
    size = torch.ldexp(torch.ones(520, device="cuda"), along if which == "late" else -1 - along).view(1, 1, -1, 1)
    if by == "key":
        v = (v.float() * size).to(T)
    else:
        do = (do.float() * size).to(T)
    _check(q, k, v, do, 1.0)


def test_a_gradient_that_is_not_finite_stays_in_its_row(gpu):
    q, k, v, do = (_rand((1, 2, 200, 64), i) for i in range(4))
    clean = _grads(q, k, v, do, causal=True)
    for spoil in (float("inf"), float("-inf"), float("nan")):
        bad = do.clone()
        bad[0, 1, 77, 5] = spoil
        got = _grads(q, k, v, bad, causal=True)
        others = [i for i in range(200) if i != 77]
        assert torch.equal(got[0][:, :, others], clean[0][:, :, others])
        assert not torch.isfinite(got[0][0, 1, 77]).any()
        for g, c in zip(got[1:], clean[1:]):
            assert torch.equal(g[:, 0], c[:, 0]) and torch.equal(g[:, 1, 78:], c[:, 1, 78:])
            assert not torch.isfinite(g[0, 1, :78, 5]).any()


@pytest.mark.parametrize("D", [32, 128, 33])
def test_values_of_small_probability(gpu, D):
    # one key takes nearly all of each row, the others some 2^-20 of it: dv of these
    # is P^T do all the same.  The bound less what it grants P in float16's steps.
    Tq, Tk = 1, 40
    q, k = _rand((1, 2, Tq, D), 1), _rand((1, 2, Tk, D), 2, 0.1)
    k[:, :, 0] = (q[:, :, 0].float() * 14.0 * math.sqrt(D) / q[:, :, 0].float().square().sum(-1, keepdim=True)).to(T)
    v, do = _rand((1, 2, Tk, D), 3), _away_from_zero(_rand((1, 2, Tq, D), 4, 2.0 ** 11), 500.0)
    value, bound = attention_64(q, k, v, False, None, None, 1 / math.sqrt(D), do)["dv"]
    bound = bound - 1.01 * STEP[T] * do.double().abs().sum(2, keepdim=True).cpu()
    assert (bound > 0).all() and (value[:, :, 1:].abs() < 2e-2).all() and (value.abs() > 6.2e-5).all()
    _within(_grads(q, k, v, do)[2], value, bound, "dv")


@pytest.mark.parametrize("Tq,Tk", [(300, 700), (2, 3000)])
@pytest.mark.parametrize("D", [64, 128, 33])
def test_the_largest_values_stay_finite(gpu, Tq, Tk, D):
    # o is a mean of v: never beyond float16's largest number, which all keys hold here
    from blitzgs_amd.attention import attention
    for seed in range(3):
        q, k = _rand((2, 4, Tq, D), seed, 3.0), _rand((2, 4, Tk, D), 10 + seed, 3.0)
        for sign in (1.0, -1.0):
            v = torch.full((2, 4, Tk, D), sign * 65504.0, device="cuda", dtype=T)
            want, bound = attention_64(q, k, v, False, None, None, 1 / math.sqrt(D))["o"]
            _within(attention(q, k, v), want, bound, "o")
            leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
            _within(attention(*leaves).detach(), want, bound, "o kept for a backward")
    # an infinity is none of these (times a probability that float16 takes for 0, it is a NaN)
    v[:, :, 5, 3] = float("inf")
    o = attention(q, k, v)
    assert not torch.isfinite(o[..., 3]).any() and torch.isfinite(o[..., 4:]).all()
