"""orthogonalise against its 64-bit form, and OrthogonalMomentum against its
formula: every type, wide, tall and square matrices of odd sides, stacks,
degenerate matrices; the refusals."""
import pytest
import torch

from token_helpers import TYPES, U, orthogonalise_64

pytestmark = pytest.mark.gpu


def _rand(shape, t, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * scale).to(t)


def _check(update, steps=5):
    from blitzgs_amd.orthogonal import orthogonalise
    got = orthogonalise(update, steps)
    assert got.shape == update.shape and got.dtype == update.dtype
    want, bound = orthogonalise_64(update, steps)
    error = torch.linalg.matrix_norm(got.double().cpu() - want)
    assert (error <= bound).all(), (error / bound).max()
    assert torch.equal(orthogonalise(update, steps), got)
    return got


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 50), (50, 1), (2, 3), (16, 16), (64, 64), (65, 63), (63, 200),
                                   (200, 63), (130, 129), (3, 40, 70), (2, 3, 33, 20), (1, 128, 500)])
def test_shapes(gpu, t, shape):
    _check(_rand(shape, t, sum(shape), 1e-2))


@pytest.mark.parametrize("t", TYPES)
def test_large_tiles(gpu, t):
    # enough tiles for the products' larger form, with sides that end inside one
    _check(_rand((16, 500, 300), t, 1))
    _check(_rand((40, 190, 400), t, 2))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", [(130, 2100), (2, 1500, 140), (200, 1100)])
def test_long_sums_of_few_tiles(gpu, t, shape):
    # the depth of X X^T is cut into parts
    _check(_rand(shape, t, 7))


@pytest.mark.parametrize("steps", [1, 2, 5, 8])
def test_steps(gpu, steps):
    _check(_rand((2, 60, 90), torch.float32, steps), steps)


def test_result_is_near_orthogonal(gpu):
    got = _check(_rand((4, 100, 300), torch.float32, 1)).double()
    s = torch.linalg.svdvals(got.cpu())
    assert s.min() > 0.6 and s.max() < 1.25


@pytest.mark.parametrize("scale", [1e-18, 1e-4, 1e4, 1e15])
def test_scales(gpu, scale):
    # the result does not depend on the scale, down to the floor under the norm
    g = _rand((40, 60), torch.float32, 3)
    _check(g * scale)


def test_zero_low_rank_and_not_finite(gpu):
    from blitzgs_amd.orthogonal import orthogonalise
    assert not orthogonalise(torch.zeros((3, 30, 40), device="cuda")).any()
    _check(_rand((30, 2), torch.float32, 1) @ _rand((2, 70), torch.float32, 2))
    g = _rand((3, 30, 40), torch.float32, 4)
    clean = orthogonalise(g)
    g[1, 2, 3] = float("nan")
    got = orthogonalise(g)
    assert torch.isnan(got[1]).all() and torch.equal(got[[0, 2]], clean[[0, 2]])


def test_strides_and_empty(gpu):
    from blitzgs_amd.orthogonal import orthogonalise
    g = _rand((50, 3, 70), torch.bfloat16, 1)
    turned = g.transpose(0, 1)
    assert torch.equal(orthogonalise(turned), orthogonalise(turned.contiguous()))
    odd = _rand((1 + 33 * 20,), torch.bfloat16, 2)[1:].view(33, 20)
    assert torch.equal(orthogonalise(odd), orthogonalise(odd.clone()))
    for shape in ((0, 4, 4), (4, 0), (2, 3, 0)):
        assert orthogonalise(torch.zeros(shape, device="cuda")).shape == shape


def test_another_stream(gpu):
    from blitzgs_amd.orthogonal import orthogonalise
    g = _rand((4, 100, 130), torch.float32, 1)
    first = orthogonalise(g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = orthogonalise(g)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(first, second)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nesterov", [True, False])
def test_optimiser_steps(gpu, t, nesterov):
    # two steps; the orthogonalised part's error is the bound above times lr,
    # the rest is two roundings of the parameter to its type
    from blitzgs_amd.orthogonal import OrthogonalMomentum
    shapes = [(40, 24), (24, 40), (40, 24), (7, 9)]
    params = [_rand(s, t, i).requires_grad_(True) for i, s in enumerate(shapes)]
    ref = [p.detach().double().cpu() for p in params]
    momenta = [torch.zeros_like(r) for r in ref]
    lr, beta, decay = 0.1, 0.9, 0.01
    opt = OrthogonalMomentum(params, lr=lr, momentum=beta, nesterov=nesterov, weight_decay=decay)
    for step in range(2):
        for i, p in enumerate(params):
            p.grad = _rand(p.shape, t, 100 * step + i)
        opt.step()
        for i, p in enumerate(params):
            g = p.grad.double().cpu()
            momenta[i] = beta * momenta[i] + g
            u = (g + beta * momenta[i] if nesterov else momenta[i]).float()
            o, bound = orthogonalise_64(u, 5)
            scale = max(1.0, p.shape[0] / p.shape[1]) ** 0.5
            ref[i] = ref[i] * (1 - lr * decay) - lr * scale * o
            off = (p.detach().double().cpu() - ref[i]).norm()
            # fp32's rounding of the momentum moves u by 4 of its steps: 4.3^5 of that in o
            assert off <= (step + 1) * (lr * scale * (bound + 1500 * 4 * U[torch.float32])
                                        + 1.1 * U[t] * ref[i].abs().norm() + 4 * U[torch.float32] * ref[i].norm())
            assert opt.state[p]["momentum_buffer"].dtype == torch.float32
            ref[i] = p.detach().double().cpu()


def test_refusals(gpu):
    from blitzgs_amd.orthogonal import OrthogonalMomentum, orthogonalise
    g = torch.zeros((4, 4), device="cuda")
    for args, words in [((g.cpu(),), "HIP device tensor"), ((g.double(),), "float32, bfloat16 or float16"),
                        ((g[0],), "matrices"), ((g, 0), "steps"), ((g, 33), "steps"), ((g, 2.0), "steps"),
                        ((torch.zeros((1, 65537), device="cuda"),), "sides")]:
        with pytest.raises(RuntimeError, match=words):
            orthogonalise(*args)
    with pytest.raises(ValueError):
        OrthogonalMomentum([g], lr=-1.0)
    with pytest.raises(ValueError):
        OrthogonalMomentum([g], lr=1.0, momentum=1.0)
    p = torch.zeros(4, device="cuda", requires_grad=True)
    p.grad = torch.zeros_like(p)
    with pytest.raises(RuntimeError, match="matrices"):
        OrthogonalMomentum([p], lr=1.0).step()
