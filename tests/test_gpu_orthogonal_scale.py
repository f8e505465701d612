"""orthogonalise at scales whose squares pass fp32's range: the result is that of
the same matrix at an ordinary scale."""
import pytest
import torch

from token_helpers import orthogonalise_64

pytestmark = pytest.mark.gpu


# in one CU; in tiles of 64 and of 128
@pytest.mark.parametrize("shape", [(40, 60), (3, 61, 39), (200, 300), (2, 300, 203), (24, 400, 500)])
@pytest.mark.parametrize("t,scale", [(torch.float32, 1e18), (torch.float32, 1e19), (torch.float32, 1e25),
                                     (torch.float32, 5e37), (torch.bfloat16, 1e25), (torch.bfloat16, 5e37)])
def test_large_matrices(gpu, shape, t, scale):
    from blitzgs_amd.orthogonal import orthogonalise
    g = torch.Generator(device="cuda").manual_seed(1)
    update = (torch.randn(shape, generator=g, device="cuda") * scale).to(t)
    if len(shape) == 3:
        update[1] = (update[1].float() / scale).to(t)     # one of the stack at an ordinary scale
    assert torch.isfinite(update).all()
    want, bound = orthogonalise_64(update, 5)
    error = torch.linalg.matrix_norm(orthogonalise(update).double().cpu() - want)
    assert (error <= bound).all(), (error / bound).max()


@pytest.mark.parametrize("shape", [(40, 60), (200, 300)])
@pytest.mark.parametrize("spoil", [float("inf"), float("-inf"), float("nan")])
def test_infinities_are_not_taken_for_large_values(gpu, shape, spoil):
    from blitzgs_amd.orthogonal import orthogonalise
    update = torch.full(shape, 1e30, device="cuda")
    update[3, 4] = spoil
    assert torch.isnan(orthogonalise(update)).all()
