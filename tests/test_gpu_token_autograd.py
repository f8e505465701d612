"""The token operators among torch's own machinery: what it cannot differentiate is
refused."""
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
