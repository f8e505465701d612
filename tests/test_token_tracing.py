"""The token operators refuse to be traced: a trace records torch's own operations, not
kernels called through their addresses, and gives unwritten memory later."""
import pytest
import torch

from blitzgs_amd.adamw import adamw_update, moment_values
from blitzgs_amd.attention import attention
from blitzgs_amd.feedforward import feed_forward
from blitzgs_amd.norm import layer_norm
from blitzgs_amd.orthogonal import orthogonalise
from blitzgs_amd.rotary import norm_rotate, rotate


def _calls(device):
    at, f = torch.arange(3, device=device), torch.ones(4, device=device, dtype=torch.int64)
    w, m = torch.ones(8, device=device), torch.ones((8, 8), device=device)
    moments = [torch.zeros(3, device=device) for _ in range(2)]
    codes, scales = torch.zeros(3, device=device, dtype=torch.uint8), torch.zeros((2, 1), device=device, dtype=torch.uint8)

    def updated(x):
        p = x.new_zeros(3)
        adamw_update([p], [torch.ones_like(p)], [moments[0]], [moments[1]], 1, 0.1)
        return p

    return [(lambda x: rotate(x, None, at, f)[0], (1, 2, 3, 8)),
            (lambda x: norm_rotate(x, x, w, w, at, f)[1], (1, 2, 3, 8)),
            (lambda x: feed_forward(x, m, m, m), (2, 8)), (lambda x: orthogonalise(x), (8, 8)), (updated, (1,)),
            (lambda x: x + moment_values(codes, codes, scales)[0], (3,)),
            (lambda x: layer_norm(x, w), (2, 8)), (lambda x: attention(x, x, x), (1, 2, 3, 8))]


@pytest.mark.parametrize("grads", [False, True])
@pytest.mark.parametrize("which", range(6))
def test_a_trace_is_refused_at_once(which, grads):
    call, shape = _calls("cpu")[which]
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(call, (torch.ones(shape, requires_grad=grads),), check_trace=False)


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(8))
def test_a_trace_is_refused(gpu, which):
    call, shape = _calls("cuda")[which]
    x = torch.ones(shape, device="cuda")
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(call, (x,), check_trace=False)
    assert torch.isfinite(call(x)).all()                # and afterwards as ever


@pytest.mark.gpu
def test_attention_is_traced_with_its_gradients(gpu):
    # it goes through an autograd function, which a trace calls again
    call, shape = _calls("cuda")[7]
    x, y = (torch.randn(shape, device="cuda", requires_grad=True) for _ in range(2))
    traced = torch.jit.trace(call, (x,), check_trace=False)
    assert torch.equal(traced(y), call(y))
