"""feed_forward against its 64-bit form: types, activations, one row to many, sizes that
end inside a tile, a chunk, a group of 16; strides; which gradients are asked for; values
at the ends of the activations; its refusals."""
import math

import pytest
import torch

from block_helpers import feed_forward_64, near
from token_helpers import TYPES, within

pytestmark = pytest.mark.gpu


def _rand(shape, t, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(t)


def _weights(W, H, O, t, seed=10):
    return (_rand((H, W), t, seed, W ** -0.5), _rand((H, W), t, seed + 1, W ** -0.5), _rand((O, H), t, seed + 2, H ** -0.5))


def _check(x, weights, activation="silu"):
    from blitzgs_amd.feedforward import feed_forward
    t = x.dtype
    leaves = [v.detach().requires_grad_(True) for v in (x, *weights)]
    y = feed_forward(*leaves, activation)
    dy = _rand(y.shape, t, 99)
    got = dict(zip(("y", "dx", "dgate", "dup", "ddown"), (y.detach(), *torch.autograd.grad(y, leaves, dy))))
    W, O = x.shape[-1], y.shape[-1]
    want = feed_forward_64(x.reshape(-1, W), *weights, activation, dy.reshape(-1, O))
    H = weights[0].shape[0]
    for name, v in got.items():
        assert v.dtype == t and v.shape == (y if name == "y" else leaves[["dx", "dgate", "dup", "ddown"].index(name)]).shape
        flat = v.reshape(want[name][0].shape)
        within(flat, *want[name], name)
        if want[name][0].numel() >= 1000:
            near(flat, want[name][0], t, max(W, 2 * H, O, x.numel() // W), name)
    with torch.no_grad():
        plain = feed_forward(x, *weights, activation)
    within(plain.reshape(want["y"][0].shape), *want["y"], "y without gradients")


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,W,H,O", [
    (1, 1, 1, 1), (1, 64, 128, 64), (3, 7, 5, 9), (17, 40, 24, 40), (130, 136, 72, 264), (64, 256, 512, 256),
    (257, 129, 131, 130), (300, 33, 517, 8), (16, 512, 264, 520), (700, 64, 16, 48)])
def test_sizes(gpu, t, activation, M, W, H, O):
    _check(_rand((M, W), t, M + W), _weights(W, H, O, t), activation)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M", [1, 2, 5, 8, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100])
def test_few_rows(gpu, t, M):
    _check(_rand((M, 264), t, M), _weights(264, 392, 200, t))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,W,H,O", [(1, 2051, 515, 301), (4, 2048, 1024, 512), (1, 8, 3000, 1100), (20, 1032, 40, 16)])
def test_few_rows_of_wide_blocks(gpu, t, M, W, H, O):
    _check(_rand((M, W), t, M), _weights(W, H, O, t))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("M", [1, 3, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("W,H,O", [(8, 256, 64), (264, 1000, 520), (2064, 2056, 72), (72, 4104, 2056), (4200, 40, 4104)])
def test_few_rows_and_columns_of_a_workgroup(gpu, t, activation, M, W, H, O):
    # 4, 8 and 16 columns to a workgroup, ends inside them and inside a step of the depth
    _check(_rand((M, W), t, M), _weights(W, H, O, t), activation)


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,W,H,O", [(2100, 320, 768, 320), (5000, 64, 64, 64), (600, 1024, 1000, 1032)])
def test_many_rows(gpu, t, M, W, H, O):
    _check(_rand((M, W), t, M), _weights(W, H, O, t))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,W,H,O", [(600, 1023, 1001, 1030), (2100, 320, 771, 320), (700, 1020, 1024, 1023), (260, 1601, 1608, 800)])
def test_large_odd_sizes(gpu, t, M, W, H, O):
    # rows that are no whole 16 bytes: of x, gate and up; of down and what lies between; of dy; of all
    wide = _rand((M, W + 5), t, 3)
    _check(wide[:, 2:W + 2], _weights(W, H, O, t))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,W,H,O", [(9, 24, 13, 24), (40, 24, 200, 24), (700, 1023, 1001, 1030)])
def test_infinite_gradients_stay_in_their_rows(gpu, t, M, W, H, O):
    from blitzgs_amd.feedforward import feed_forward
    x, weights, dy = _rand((M, W), t, 1).requires_grad_(True), _weights(W, H, O, t), _rand((M, O), t, 2)
    (clean,) = torch.autograd.grad(feed_forward(x, *weights), x, dy)
    dy[3, 0] = dy[5, O - 1] = math.inf
    (g,) = torch.autograd.grad(feed_forward(x, *weights), x, dy)
    rows = [r for r in range(M) if r not in (3, 5)]
    assert torch.equal(g[rows], clean[rows]) and not torch.isfinite(g[[3, 5]]).any()


@pytest.mark.parametrize("t", TYPES)
def test_strides_and_dimensions(gpu, t):
    from blitzgs_amd.feedforward import feed_forward
    W, H, O = 64, 96, 64
    weights = _weights(W, H, O, t)
    wide = _rand((50, 3 * W + 8), t, 1)
    _check(wide[:, 8:8 + W], weights)                               # whole chunks, rows apart
    _check(wide[:, 3:3 + W], weights)                               # rows that start off 16 bytes
    _check(_rand((W, 50), t, 2).t(), weights)                       # the last dimension not contiguous
    _check(_rand((2, 5, 7, W), t, 3), weights)                      # more dimensions
    _check(_rand((W,), t, 4), weights)                              # one row of one dimension
    _check(_rand((1, W), t, 5).expand(20, W), weights)              # one row for all
    turned = [w.t().contiguous().t() for w in weights]              # weights that lie transposed
    _check(_rand((33, W), t, 6), turned)
    off = [_rand((w.numel() + 1,), t, 7)[1:].view(w.shape).copy_(w) for w in weights]   # and off 16 bytes
    _check(_rand((33, W), t, 8), off)
    # a broadcast gradient, and one whose rows lie apart
    x = _rand((40, W), t, 9).requires_grad_(True)
    y = feed_forward(x, *weights)
    (a,) = torch.autograd.grad(y, x, torch.ones((), device="cuda", dtype=t).expand(y.shape), retain_graph=True)
    (b,) = torch.autograd.grad(y, x, torch.ones((40, 2 * O), device="cuda", dtype=t)[:, O:], retain_graph=True)
    (c,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(a, c) and torch.equal(b, c)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_rows_far_apart_and_very_many(gpu, t):
    # rows of 4 million elements each: a tile of them spans more than a 32-bit offset is used for
    far = torch.empty((20, (1 << 22) + 8), device="cuda", dtype=t)[:, :64]
    far.copy_(_rand((20, 64), t, 1))
    _check(far, _weights(64, 72, 40, t))
    _check(_rand((70001, 24), t, 2), _weights(24, 40, 16, t))


@pytest.mark.parametrize("t", TYPES)
def test_which_gradients_are_asked_for(gpu, t):
    from blitzgs_amd.feedforward import feed_forward
    args = [_rand((70, 48), t, 1), *_weights(48, 80, 56, t)]
    dy = _rand((70, 56), t, 5)
    leaves = [a.clone().requires_grad_(True) for a in args]
    every = torch.autograd.grad(feed_forward(*leaves), leaves, dy)
    for asked in ((0,), (1,), (2,), (3,), (0, 3), (1, 2)):
        leaves = [a.clone().requires_grad_(i in asked) for i, a in enumerate(args)]
        got = torch.autograd.grad(feed_forward(*leaves), [leaves[i] for i in asked], dy)
        assert all(torch.equal(a, every[i]) for i, a in zip(asked, got))


def test_no_rows(gpu):
    from blitzgs_amd.feedforward import feed_forward
    leaves = [torch.empty((0, 8), device="cuda", requires_grad=True)]
    leaves += [w.requires_grad_(True) for w in _weights(8, 16, 8, torch.float32)]
    y = feed_forward(*leaves)
    assert y.shape == (0, 8)
    y.sum().backward()
    assert leaves[0].grad.shape == (0, 8)
    assert all(torch.equal(w.grad, torch.zeros_like(w)) for w in leaves[1:])


@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_the_ends_of_the_activations(gpu, activation):
    # projections that copy: a = b = x; up to where exp overflows
    from blitzgs_amd.feedforward import feed_forward
    x = torch.tensor([-200.0, -90.0, -30.0, -9.0, -4.0, -1e-3, 0.0, 1e-3, 4.0, 9.0, 30.0, 200.0], device="cuda")
    eye = torch.eye(12, device="cuda")
    leaf = x[None].clone().requires_grad_(True)
    y = feed_forward(leaf, eye, eye, eye, activation)
    (g,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    want = feed_forward_64(x[None], eye, eye, eye, activation, torch.ones((1, 12)))
    within(y, *want["y"], "y")
    within(g, *want["dx"], "dx")


@pytest.mark.parametrize("M", [1, 4, 7, 16])
@pytest.mark.parametrize("W,H,O", [(12, 20, 28), (1028, 516, 132), (2044, 1024, 260), (4, 4, 4), (8, 1028, 64), (64, 65, 64)])
def test_few_rows_of_whole_pieces_of_four(gpu, M, W, H, O):
    # float: 16 bytes are four elements, of which a depth may end half way in a lane's eight; what lies behind x is
    # not a number
    wide = torch.full((M, W + 4), math.nan, device="cuda")
    wide[:, :W] = _rand((M, W), torch.float32, M)
    _check(wide[:, :W], _weights(W, H, O, torch.float32))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M", [3, 8, 13])
def test_nan_stays_in_its_row_of_few(gpu, t, M):
    from blitzgs_amd.feedforward import feed_forward
    x, weights = _rand((M, 200), t, 1), _weights(200, 520, 264, t)
    clean = feed_forward(x, *weights)
    for bad in (math.nan, math.inf):
        y = x.clone()
        y[1, 0] = y[1, 199] = bad
        got = feed_forward(y, *weights)
        others = [i for i in range(M) if i != 1]
        assert got[1].isnan().any() and torch.equal(got[others], clean[others])


def test_nan_stays_in_its_row(gpu):
    from blitzgs_amd.feedforward import feed_forward
    for M in (9, 300):
        x, weights = _rand((M, 72), torch.bfloat16, 1), _weights(72, 80, 64, torch.bfloat16)
        clean = feed_forward(x, *weights)
        x[4, 7] = float("nan")
        x[5, 3] = float("inf")
        y = feed_forward(x, *weights)
        assert torch.isnan(y[4]).all() and not torch.isfinite(y[5]).any()
        rows = [r for r in range(M) if r not in (4, 5)]
        assert torch.equal(y[rows], clean[rows])


def test_gradient_against_differences(gpu):
    # f = sum(y c): central differences along a random direction in fp32, steps of 1e-2: a truncation error of
    # the order of 1e-4 of the derivative's size and noise far below 1e-2
    from blitzgs_amd.feedforward import feed_forward
    args = [_rand((20, 24), torch.float32, 0), *_weights(24, 40, 16, torch.float32)]
    c = _rand((20, 16), torch.float32, 9)
    for activation in ("silu", "gelu"):
        f = lambda *a: (feed_forward(*a, activation).double() * c.double()).sum().item()  # noqa: E731, B023
        leaves = [p.clone().requires_grad_(True) for p in args]
        grads = torch.autograd.grad(feed_forward(*leaves, activation), leaves, c)
        for i in range(4):
            d = _rand(args[i].shape, torch.float32, 20 + i)
            d /= d.norm()
            up, down = list(args), list(args)
            up[i], down[i] = args[i] + 1e-2 * d, args[i] - 1e-2 * d
            along = (grads[i].double() * d.double()).sum().item()
            assert abs((f(*up) - f(*down)) / 2e-2 - along) <= 1e-2 * (1 + abs(along))


@pytest.mark.parametrize("M", [3, 2000])
def test_equal_bits_and_another_stream(gpu, M):
    from blitzgs_amd.feedforward import feed_forward
    args = [_rand((M, 256), torch.bfloat16, 1), *_weights(256, 512, 256, torch.bfloat16)]

    def once():
        leaves = [a.clone().requires_grad_(True) for a in args]
        y = feed_forward(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, args[0])]

    first = once()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = once()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_refusals(gpu):
    from blitzgs_amd.feedforward import feed_forward
    x = torch.zeros((4, 8), device="cuda")
    gate, up, down = _weights(8, 16, 8, torch.float32)
    for args, words in [((x.double(), gate, up, down), "float32, bfloat16 or float16"),
                        ((x.cpu(), gate, up, down), "HIP device tensor"),
                        ((x, gate.bfloat16(), up, down), "gate must be"), ((x, gate, up[0], down), "up must be"),
                        ((x, gate, up, down.cpu()), "HIP device tensor"), ((x[:, :7], gate, up, down), "for x"),
                        ((x, gate, up[:15], down), "for x"), ((x, gate, up, down[:, :15]), "for x"),
                        ((x, gate[:0], up[:0], down[:, :0]), "sides of 1"), ((x, gate, up, down, "relu"), "activation")]:
        with pytest.raises(RuntimeError, match=words):
            feed_forward(*args)
    assert math.isfinite(feed_forward(x, gate, up, down).sum().item())
