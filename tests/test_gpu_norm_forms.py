"""layer_norm in 16-byte accesses from rows that start off 16 bytes, and the
partial sums of squares of orthogonalise where its matrices do."""
import pytest
import torch

from token_helpers import TYPES, layer_norm_64, orthogonalise_64, within

pytestmark = pytest.mark.gpu


def _rand(shape, t, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("width", [8, 64, 520, 1024, 4096])
@pytest.mark.parametrize("apart", [1, 3, 8])
def test_whole_accesses_at_odd_addresses(gpu, t, width, apart):
    from blitzgs_amd.norm import layer_norm
    rows = 37
    wide = lambda seed: _rand((rows * (width + apart) + 1,), t, seed)[1:].view(rows, width + apart)[:, :width]  # noqa
    x, dy = wide(1), wide(2)
    w, b = _rand((width + 1,), t, 3)[1:], _rand((width + 1,), t, 4)[1:]
    leaves = [p.detach().requires_grad_(True) for p in (x, w, b)]
    y = layer_norm(*leaves)
    got = dict(zip(("y", "dx", "dweight", "dbias"), (y.detach(), *torch.autograd.grad(y, leaves, dy))))
    want = layer_norm_64(x, w, b, 1e-5, dy, rows_chain=rows)
    for name in got:
        within(got[name], *want[name], name)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", [(3, 201, 203), (2, 131, 1001)])
def test_stacks_of_odd_matrices(gpu, t, shape):
    from blitzgs_amd.orthogonal import orthogonalise
    update = _rand(shape, t, 1)
    want, bound = orthogonalise_64(update, 5)
    error = torch.linalg.matrix_norm(orthogonalise(update).double().cpu() - want)
    assert (error <= bound).all(), (error / bound).max()
