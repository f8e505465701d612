"""norm_rotate of rows whose squares fp32 does not hold, alone and among ordinary rows."""
import math

import pytest
import torch

from block_helpers import rotary_64
from token_helpers import TYPES, within

pytestmark = pytest.mark.gpu


def _rand(shape, t, seed, scale=1.0, mean=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale + mean).to(t)


def _check(q, k, w, eps, interleaved, pairs):
    from blitzgs_amd.rotary import norm_rotate, rotary_frequencies
    at, f = torch.arange(q.shape[2], device="cuda"), rotary_frequencies(pairs)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, w)]
    outs = norm_rotate(leaves[0], leaves[1], leaves[2], None, at, f, interleaved, eps=eps)
    grads = [_rand(o.shape, q.dtype, 90 + i) for i, o in enumerate(outs)]
    dq, dk, dw = torch.autograd.grad(outs, leaves, grads)
    for out, dx, x, weight, dy, name in ((outs[0], dq, q, w, grads[0], "q"), (outs[1], dk, k, None, grads[1], "k")):
        want = rotary_64(x, weight, dy, at, f, interleaved, 1.0, True, eps)
        within(out, *want["y"], name)
        value, bound = want["dx"]
        there = value.abs() < torch.finfo(q.dtype).max
        within(dx.cpu()[there], value[there], bound[there], "d" + name)
        if weight is not None:
            within(dw, *want["dw"], "dw")


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D,pairs", [(64, 32), (75, 35), (129, 64), (16, 4), (2, 1)])
@pytest.mark.parametrize("size", [1e17, 1e19, 1e25, 1e30, 4e37])
def test_large_rows(gpu, t, size, D, pairs, interleaved):
    q, k, w = _rand((2, 3, 7, D), t, 1, 1.5), _rand((2, 2, 7, D), t, 2), _rand((D,), t, 3, 0.2, 1.0)
    _check(q * size, k * size, w, 1e-6, interleaved, pairs)
    # one row of many, and one element of a row
    one, two = q.clone(), k.clone()
    one[1, 2, 3] *= size
    two[0, 1, 6, D - 1] = size
    _check(one, two, w, 1e-6, interleaved, pairs)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D,pairs", [(64, 32), (75, 35)])
@pytest.mark.parametrize("eps", [0.0, 1e-38])
@pytest.mark.parametrize("size", [1e-14, 1e-19, 1e-22, 1e-30, 1e-36])
def test_small_rows_with_little_or_no_eps(gpu, t, size, eps, D, pairs):
    q, k, w = _rand((2, 3, 7, D), t, 1, 1.5), _rand((2, 2, 7, D), t, 2), _rand((D,), t, 3, 0.2, 1.0)
    _check((q.float() * size).to(t), (k.float() * size).to(t), w, eps, True, pairs)
    one = q.clone()
    one[1, 2, 3] *= size
    _check(one, k, w, eps, False, pairs)


@pytest.mark.parametrize("t", TYPES)
def test_a_large_eps_and_no_number(gpu, t):
    from blitzgs_amd.rotary import norm_rotate, rotary_frequencies
    q, w = _rand((1, 2, 5, 32), t, 1), _rand((32,), t, 3)
    _check(q, q[:, :1], w, 1e38, False, 8)
    at, f = torch.arange(5, device="cuda"), rotary_frequencies(8)
    clean = norm_rotate(q, None, w, None, at, f)[0]
    for bad in (math.nan, math.inf):
        x = q.clone()
        x[0, 1, 2, 5] = bad
        y = norm_rotate(x, None, w, None, at, f)[0]
        assert y[0, 1, 2, 5].isnan()
        y[0, 1, 2] = clean[0, 1, 2]
        assert torch.equal(y, clean)
