"""layer_norm against its 64-bit form: every type, rows of one to many, widths
that end inside a 16-byte chunk, a wave, a block; strides; its refusals."""
import pytest
import torch

from token_helpers import TYPES, layer_norm_64, within

pytestmark = pytest.mark.gpu

EPS = 1e-5


def _rand(shape, t, seed, scale=1.0, mean=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale + mean).to(t)


def _check(x, w, b, dy, eps=EPS):
    from blitzgs_amd.norm import layer_norm
    leaves = [None if p is None else p.detach().requires_grad_(True) for p in (x, w, b)]
    # a view's gradient is asked for at the view
    y = layer_norm(*leaves, eps)
    asked = [p for p in leaves if p is not None]
    grads = dict(zip([n for n, p in zip(("dx", "dweight", "dbias"), leaves) if p is not None],
                     torch.autograd.grad(y, asked, dy)))
    rows = x.numel() // x.shape[-1]
    want = layer_norm_64(x, w, b, eps, dy, rows_chain=rows)
    assert y.dtype == x.dtype and y.shape == x.shape
    within(y, *want["y"], "y")
    for name, got in grads.items():
        within(got, *want[name], name)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps), y.detach())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (1, 64), (257, 33), (5, 256), (700, 513), (33, 1024),
                                        (9, 2049), (4, 4100), (3, 8200), (2, 32768)])
def test_rows_and_widths(gpu, t, rows, width):
    x, dy = _rand((rows, width), t, rows + width, 1.5, 0.3), _rand((rows, width), t, 1)
    _check(x, _rand((width,), t, 2, 0.2, 1.0), _rand((width,), t, 3, 0.2), dy)


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
def test_parameters_in_32_bits_and_absent(gpu, t):
    x, dy = _rand((65, 200), t, 1), _rand((65, 200), t, 2)
    w, b = _rand((200,), torch.float32, 3, 0.2, 1.0), _rand((200,), torch.float32, 4)
    for params in ((w, b), (w, None), (None, b), (None, None)):
        _check(x, *params, dy)


def test_offsets_of_the_mean(gpu):
    # a row's mean far above its spread: a one-pass variance would lose it
    x = _rand((40, 300), torch.float32, 1, 1e-2, 50.0)
    _check(x, None, None, _rand((40, 300), torch.float32, 2))


@pytest.mark.parametrize("t", TYPES)
def test_strided_and_odd_addresses(gpu, t):
    wide = _rand((50, 3 * 65 + 1), t, 1)
    dy = _rand((50, 65), t, 2)
    _check(wide[:, 66:131], None, None, dy)                                # a slice that starts off 16 bytes
    _check(_rand((65, 50), t, 3).t(), None, None, dy)                      # the last dimension not contiguous
    _check(_rand((1, 65), t, 4).expand(50, 65), None, None, dy)            # one row for all
    _check(_rand((5, 10, 65), t, 5), None, None, dy.view(5, 10, 65))       # more dimensions
    _check(_rand((50, 65), t, 6), None, None, _rand((65,), t, 7).expand(50, 65))   # a broadcast gradient


def test_constant_rows_and_no_rows(gpu):
    from blitzgs_amd.norm import layer_norm
    x = torch.full((4, 96), 3.0, device="cuda", requires_grad=True)
    y = layer_norm(x)
    assert torch.equal(y, torch.zeros_like(y))
    (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.isfinite(g).all()
    w = torch.ones(96, device="cuda", requires_grad=True)
    e = torch.empty((0, 96), device="cuda", requires_grad=True)
    y = layer_norm(e, w, w)
    assert y.shape == (0, 96)
    y.sum().backward()
    assert torch.equal(w.grad, torch.zeros_like(w)) and e.grad.shape == (0, 96)


def test_nan_stays_in_its_row(gpu):
    from blitzgs_amd.norm import layer_norm
    x = _rand((9, 130), torch.float32, 1)
    clean = layer_norm(x)
    x[4, 7] = float("nan")
    y = layer_norm(x)
    assert torch.isnan(y[4]).all()
    rows = [r for r in range(9) if r != 4]
    assert torch.equal(y[rows], clean[rows])


def test_gradient_against_differences(gpu):
    # f = sum(y c): central differences along a random direction, in fp32; the
    # step of 1e-2 leaves a truncation error of about 1e-4 of the derivative's
    # size and a noise of sqrt(n) 2^-24 / 1e-2, both far below 1e-2
    from blitzgs_amd.norm import layer_norm
    x, w, b = (_rand(s, torch.float32, i) for i, s in enumerate([(20, 48), (48,), (48,)]))
    c = _rand((20, 48), torch.float32, 9)
    f = lambda *a: (layer_norm(*a).double() * c.double()).sum().item()  # noqa: E731
    leaves = [p.clone().requires_grad_(True) for p in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, c)
    for i in range(3):
        d = _rand(leaves[i].shape, torch.float32, 20 + i)
        d /= d.norm()
        h = 1e-2
        up, down = [x, w, b], [x, w, b]
        up[i], down[i] = up[i] + h * d, down[i] - h * d
        along = (grads[i].double() * d.double()).sum().item()
        assert abs((f(*up) - f(*down)) / (2 * h) - along) <= 1e-2 * (1 + abs(along))


def test_equal_bits_and_another_stream(gpu):
    from blitzgs_amd.norm import layer_norm
    x, dy = _rand((5000, 520), torch.bfloat16, 1), _rand((5000, 520), torch.bfloat16, 2)
    w = _rand((520,), torch.float32, 3)

    def once():
        leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
        y = layer_norm(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    first = once()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = once()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_refusals(gpu):
    from blitzgs_amd.norm import layer_norm
    x = torch.zeros((4, 8), device="cuda")
    w = torch.ones(8, device="cuda")
    for bad, words in [((x.double(),), "float32, bfloat16 or float16"), ((x.cpu(),), "HIP device tensor"),
                       ((x, w[:7]), r"shape \(8,\)"), ((x, w.bfloat16()), "weight must be"),
                       ((x.bfloat16(), w, w.bfloat16()), "one type"), ((x, w.cpu()), "HIP device tensor"),
                       ((x, None, None, -1.0), "eps"), ((torch.zeros((2, 0), device="cuda"),), "last dimension"),
                       ((torch.zeros((1, 32769), device="cuda"),), "last dimension")]:
        with pytest.raises(RuntimeError, match=words):
            layer_norm(*bad)
