"""feed_forward at the ends of its types' ranges: projections beyond float16's largest
number, whose products and gradients are within it; the activations' ends in 16 bits."""
import math

import pytest
import torch

from block_helpers import feed_forward_64
from token_helpers import U, U32, within

pytestmark = pytest.mark.gpu


def _rand(shape, t, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(t)


def _grads(args, dy, activation):
    from blitzgs_amd.feedforward import feed_forward
    leaves = [v.detach().requires_grad_(True) for v in args]
    y = feed_forward(*leaves, activation)
    return dict(zip(("y", "dx", "dgate", "dup", "ddown"), (y.detach(), *torch.autograd.grad(y, leaves, dy))))


# few rows, small tiles, odd sizes, large tiles, large tiles of copies
@pytest.mark.parametrize("M,W,H,O", [(1, 16, 24, 16), (5, 264, 512, 256), (60, 33, 71, 40), (300, 64, 128, 64),
                                     (2100, 320, 768, 320), (700, 1023, 1001, 1030)])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("large", ["gate", "up"])
def test_projections_beyond_float16(gpu, large, t, activation, M, W, H, O):
    # half of x's columns make a, the other half b; one of the two is of the order of 1e5, the other of 0.05
    half = W // 2
    x, dy = _rand((M, W), t, 1), _rand((M, O), t, 2, 0.01)
    weights = [torch.zeros((H, W), device="cuda", dtype=t) for _ in range(2)]
    for w, columns, big, seed in ((weights[0], slice(0, half), large == "gate", 3),
                                  (weights[1], slice(half, W), large == "up", 4)):
        n = columns.stop - columns.start
        w[:, columns] = _rand((H, n), t, seed, (500 if big else 0.05) / math.sqrt(n))
        if big:
            x[:, columns] *= 200
    args = (x, *weights, _rand((O, H), t, 5, H ** -0.5))
    got = _grads(args, dy, activation)
    want = feed_forward_64(x, *args[1:], activation, dy)
    if t == torch.float16:
        assert ((x.double() @ weights[large == "up"].double().T).abs() > 65504).double().mean() > 0.2
    within(got["y"], *want["y"], "y")
    for name in ("dx", "dgate", "dup", "ddown"):
        g, (w, bound) = got[name].double().cpu(), want[name]
        # The bound holds a rounding of da and db to the type, 2^-11; a or b beyond 65504 may be off by 2^-8, of which
        # the activation makes 1.13 times that: nine times as much again.  A sum that is itself beyond float16's range,
        # or may be, is left out: up's gradient where x is as large as it is for the gate
        loose = 10 * bound if t == torch.float16 else bound
        there = w.abs() + loose < 65504 if t == torch.float16 else torch.ones_like(w, dtype=torch.bool)
        assert there.double().mean() > 0.3 and not g.isnan().any(), name
        within(g[there], w[there], loose[there], name)
        if there.all():
            # as elsewhere up to four roundings to the type, and the one to 2^-8
            rel = ((g - w).norm() / w.norm()).item()
            most = 2 * U[t] + (2.0 ** -8 if t == torch.float16 else 0) + 4 * math.sqrt(max(W, 2 * H, O, M) + 16) * U32
            assert rel <= most, (name, rel)


@pytest.mark.parametrize("rows", [1, 4, 20])
def test_the_border_of_float16(gpu, rows):
    # a = 65504 + c, which float16 rounds to 65504 up to 65519
    c = torch.tensor([0.0, 8.0, 15.5, 15.99, 16.0, 17.0, 100.0, 30000.0, 60000.0], device="cuda").half()
    n = len(c)
    x = torch.tensor([[65504.0, 1.0]], device="cuda").half().expand(rows, 2).contiguous()
    gate = torch.stack([torch.ones_like(c), c], 1)
    up = torch.tensor([0.0, 0.25], device="cuda").half().expand(n, 2).contiguous()
    down = torch.eye(n, device="cuda").half()
    dy = torch.full((rows, n), 2.0 ** -6, device="cuda").half()
    got = _grads((x, gate, up, down), dy, "silu")
    a = 65504.0 + c.double().cpu()
    # one rounding of a kept number, 2^-8 beyond the border and 2^-14 below it, and float16's two of a result
    loose = torch.where(a >= 65520, 2.0 ** -8, 2.0 ** -14) + 2 * 2.0 ** -11
    dup = 2.0 ** -6 * a * rows
    assert ((got["dup"][:, 1].double().cpu() - dup).abs() <= loose * dup).all()
    dx = 0.25 * 2.0 ** -6 * a.sum()
    assert ((got["dx"][:, 1].double().cpu() - dx - 2.0 ** -6 * 0.25 * c.double().cpu().sum()).abs() <= loose.max() * 2 * dx).all()
    # a's own gradient is exact
    assert torch.equal(got["dgate"][:, 1], torch.full_like(c, 2.0 ** -6 * 0.25 * rows))


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_the_ends_of_the_activations_in_16_bits(gpu, activation, t):
    # projections that copy: a = b = x; down to float16's subnormals
    x = torch.tensor([-200.0, -90.0, -30.0, -16.0, -9.0, -4.0, -1e-3, -2e-5, -1e-6, 0.0, 6e-8, 1e-6, 2e-5, 1e-3, 4.0, 9.0,
                      16.0, 30.0, 200.0, 250.0], device="cuda").to(t)
    n = len(x)
    eye = torch.eye(n, device="cuda", dtype=t)
    for rows in (1, 40):
        xs = x[None].expand(rows, n).contiguous()
        dy = torch.ones((rows, n), device="cuda", dtype=t)
        got = _grads((xs, eye, eye, eye), dy, activation)
        want = feed_forward_64(xs, eye, eye, eye, activation, dy)
        within(got["y"], *want["y"], "y")
        within(got["dx"], *want["dx"], "dx")


@pytest.mark.parametrize("rows", [1, 40])
def test_what_rounding_left_of_projections_of_all_sizes(gpu, rows):
    # a = x (1 + c 2^-12): float16 rounds its last two bits away, the rest keeps them
    x = torch.tensor([1000.0, 130.0, 3.0, 1.0, 2.0 ** -10, 2.0 ** -13], device="cuda").half()
    n = len(x)
    gate, up = torch.zeros((n, 2 * n), device="cuda").half(), torch.zeros((n, 2 * n), device="cuda").half()
    gate[:, :n] = gate[:, n:] = torch.eye(n, device="cuda").half()
    up[:, n:] = 0.25 * torch.eye(n, device="cuda").half()
    wide = torch.cat([x, (x.double() * 2.0 ** -12).half()])[None].expand(rows, 2 * n).contiguous()
    eye = torch.eye(n, device="cuda").half()
    dy = torch.full((rows, n), 0.125, device="cuda").half()
    got = _grads((wide, gate, up, eye), dy, "gelu")
    want = feed_forward_64(wide, gate, up, eye, "gelu", dy)
    for name in ("y", "dx"):
        within(got[name], *want[name], name)
