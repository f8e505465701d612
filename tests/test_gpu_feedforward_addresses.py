"""feed_forward of large blocks whose sizes are whole 16 bytes and whose addresses or
strides are not: x and its gradient as slices, weights in one flat buffer."""
import pytest
import torch

from block_helpers import feed_forward_64, near
from token_helpers import TYPES, within

pytestmark = pytest.mark.gpu


def _rand(shape, t, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("off", ["x", "dy", "weights", "all"])
@pytest.mark.parametrize("M,W,H,O", [(300, 1024, 1032, 1024), (260, 1027, 1024, 1000)])
def test_odd_addresses(gpu, t, off, M, W, H, O):
    from blitzgs_amd.feedforward import feed_forward
    x, dy = _rand((M, W), t, 1), _rand((M, O), t, 2)
    shapes = [(H, W), (H, W), (O, H)]
    weights = [_rand(s, t, 3 + i, s[1] ** -0.5) for i, s in enumerate(shapes)]
    if off in ("x", "all"):
        x = torch.cat([x[:, :3], x, x[:, :2]], 1)[:, 3:3 + W]
    if off in ("dy", "all"):
        dy = torch.cat([dy[:, :1], dy, dy[:, :4]], 1)[:, 1:1 + O]
    if off in ("weights", "all"):
        flat = torch.cat([w.flatten() for w in [weights[0][0, :1], *weights]])
        weights = [p.view(s) for p, s in zip(flat[1:].split([a * b for a, b in shapes]), shapes)]
    leaves = [v.detach().requires_grad_(True) for v in (x, *weights)]
    y = feed_forward(*leaves)
    got = dict(zip(("y", "dx", "dgate", "dup", "ddown"), (y.detach(), *torch.autograd.grad(y, leaves, dy))))
    want = feed_forward_64(x, *weights, "silu", dy)
    for name, v in got.items():
        within(v, *want[name], name)
        near(v, want[name][0], t, max(W, 2 * H, O, M), name)
