"""8-bit moments over many steps beside AdamW's own: blocks of elements whose gradients are
of very different sizes; moments next to the largest number there is."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BLOCK = 128


def _sizes(kind, n):
    """How large the gradients of n elements are, and which are quiet: a thousandth of their block's largest or less."""
    if kind == "log-normal":
        size = torch.exp(2 * torch.randn(n, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda"))
    else:
        size = torch.full((n,), kind, device="cuda")
        size.view(-1, BLOCK)[:, 3:11] = 1.0
    largest = size.view(-1, BLOCK).amax(1).repeat_interleave(BLOCK)
    return size, size <= 1e-3 * largest


@pytest.mark.parametrize("constant", [False, True])
@pytest.mark.parametrize("kind", [1e-4, 1e-5, 1e-6, 1e-8, "log-normal"])
def test_quiet_elements_of_a_loud_block(gpu, kind, constant):
    # An update over lr is at most c1 / sqrt(c2 (1 - b1^2 / b2)) = 7.3 whatever the gradients (Cauchy and Schwarz; the
    # corrections of the first steps only shrink it).  Rounding moves m by less than a step each time, and 0.9^k of that
    # is left k steps later: less than 9 steps in all.  A step is an eighth of m, or 2^-16 of the power of two of the
    # block's largest m, which is at most the root of the block's largest v for gradients of alternating or of one
    # sign; and v's root is never below 2^-16 of that of its block's power of two, 1 / sqrt(2) of the largest's root or
    # more.  So no update is above 7.3 + 9 sqrt(2) = 20.  On average a rounding has a variance of at most a quarter of a
    # step's square, all that are left of them together 1 / (1 - 0.81) times that, 1.15 steps: 1.15 sqrt(2) = 1.6, and
    # at most 1 of the update itself
    from blitzgs_amd.adamw import adamw_update, new_moments
    n, steps = 32 * BLOCK, 400
    size, quiet = _sizes(kind, n)
    p = torch.zeros(n, device="cuda")
    m, v, s = new_moments(p, 8)
    largest, square = 0.0, torch.zeros(n, device="cuda", dtype=torch.float64)
    rng = torch.Generator(device="cuda").manual_seed(6)
    for k in range(steps):
        g = size if constant else size * torch.randn(n, generator=rng, device="cuda").sign()
        p.zero_()
        adamw_update([p], [g], [m], [v], step=k + 1, lr=1.0, weight_decay=0.0, scales=[s])
        largest = max(largest, p.abs().max().item())
        square += p.double().square()
    assert largest <= 7.3 + 9 * math.sqrt(2)
    assert (square[quiet] / steps).mean().sqrt().item() <= 1 + 1.15 * math.sqrt(2)
    # a second moment that is not zero is not forgotten
    assert (v[size > 0] > 0).all()


@pytest.mark.parametrize("seed", range(6))
def test_moments_next_to_the_largest_number(gpu, seed):
    # 1.97 2^127 lies between the code of 1.875 2^127 and that of 2^128, which is no number: it is never rounded up
    from blitzgs_amd.adamw import adamw_update, moment_values, new_moments
    top = 1.97 * 2.0 ** 127
    for moment, g, betas in ((0, top, (0.0, 0.999)), (0, -top, (0.0, 0.999)), (1, math.sqrt(top), (0.0, 0.0))):
        p = torch.zeros(300, device="cuda")
        m, v, s = new_moments(p, 8)
        adamw_update([p], [torch.full_like(p, g)], [m], [v], step=1, lr=0.0, betas=betas, weight_decay=0.0, scales=[s],
                     seed=seed)
        got = moment_values(m, v, s)[moment]
        assert torch.equal(got, torch.full_like(got, math.copysign(1.875 * 2.0 ** 127, g)))
