"""The token operators among torch's own machinery: what it cannot differentiate is
refused, and what it has to know of is told."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def _rand(shape, seed, t=torch.float32):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(t)


# neither operator has a forward-mode derivative: a tangent is refused, not dropped
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("also_backward", [False, True])
@pytest.mark.parametrize("grad_mode", [False, True])
def test_a_forward_mode_tangent_is_refused(gpu, which, also_backward, grad_mode):
    from blitzgs_amd.attention import attention
    from blitzgs_amd.norm import layer_norm
    norm = [_rand((5, 16), 0), _rand((16,), 1), _rand((16,), 2)]
    attn = [_rand((1, 2, 4, 16), i) for i in range(3)]
    for op, args in ((layer_norm, norm), (attention, attn)):
        if also_backward:
            args = [a.requires_grad_(True) for a in args]
        with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
            op(*args)                                       # without a tangent: as ever
            args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
            with pytest.raises(NotImplementedError, match="jvp|forward"):
                op(*args)


def test_a_step_is_seen_by_graphs_that_hold_the_weights(gpu):
    # as with torch's own optimisers: what saved a weight before the step cannot be differentiated after it
    from blitzgs_amd.orthogonal import OrthogonalMomentum
    for t in (torch.float32, torch.bfloat16):
        w = _rand((24, 16), 0, t).requires_grad_(True)
        opt = OrthogonalMomentum([w], lr=0.1)
        x = _rand((5, 16), 1, t).requires_grad_(True)
        y = x @ w.t()
        w.grad = torch.ones_like(w)
        opt.step()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
        (x @ w.t()).sum().backward()                        # a new graph is fine
