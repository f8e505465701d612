"""rotate and norm_rotate against their 64-bit forms: types, layouts, axes, heads that
share keys, one token to many, odd heads, far and negative positions, strides; their
gradients against differences; their refusals."""
import math

import pytest
import torch

from block_helpers import rotary_64
from token_helpers import TYPES, within

pytestmark = pytest.mark.gpu


def _rand(shape, t, seed, scale=1.0, mean=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale + mean).to(t)


def _check(q, k, qw, kw, positions, frequencies, interleaved=False, magnitude=1.0, norm=True, eps=1e-6):
    from blitzgs_amd.rotary import norm_rotate, rotate
    t = q.dtype
    leaves = [None if x is None else x.detach().requires_grad_(True) for x in (q, k, qw, kw)]

    def call(q, k, qw, kw):
        if norm:
            return norm_rotate(q, k, qw, kw, positions, frequencies, interleaved, magnitude, eps)
        return rotate(q, k, positions, frequencies, interleaved, magnitude)

    outs = call(*leaves)
    assert (outs[1] is None) == (k is None)
    outs = [o for o in outs if o is not None]
    grads = [_rand(o.shape, t, 90 + i) for i, o in enumerate(outs)]
    asked = [x for x in leaves if x is not None]
    got = dict(zip([n for n, x in zip(("dq", "dk", "dqw", "dkw"), leaves) if x is not None],
                   torch.autograd.grad(outs, asked, grads)))
    for i, (x, w, side) in enumerate(((q, qw, "q"), (k, kw, "k"))):
        if x is None:
            continue
        want = rotary_64(x, w, grads[i], positions, frequencies, interleaved, magnitude, norm, eps)
        assert outs[i].dtype == t and outs[i].shape == x.shape
        within(outs[i], *want["y"], side)
        within(got["d" + side], *want["dx"], "d" + side)
        if w is not None:
            assert got[f"d{side}w"].dtype == w.dtype
            within(got[f"d{side}w"], *want["dw"], f"d{side}w")
    with torch.no_grad():
        for a, b in zip([o for o in call(q, k, qw, kw) if o is not None], outs):
            assert torch.equal(a, b.detach())


def _frequencies(pairs, axes=1, base=10000.0):
    from blitzgs_amd.rotary import rotary_frequencies
    return rotary_frequencies(pairs, base=base, axes=axes)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("B,Hq,Hk,T,D,pairs", [
    (1, 1, 1, 1, 2, 1),            # the least there is
    (2, 4, 2, 9, 64, 32),          # whole accesses
    (3, 5, 1, 33, 128, 32),        # half of the head
    (2, 3, 3, 17, 75, 35),         # odd heads: items of fewer
    (1, 2, 1, 5, 40, 20),          # accesses of 8 bytes
    (1, 2, 2, 3, 256, 128),        # the widest
    (1, 3, 2, 4, 255, 127),        # the widest odd ones
    (2, 6, 2, 700, 32, 16),        # many tokens
    (5, 1, 1, 3, 96, 16),
    (1, 300, 1, 2, 16, 8),         # more heads than groups of lanes
    (1, 1, 1, 2, 7, 1)])
def test_sizes(gpu, t, norm, interleaved, B, Hq, Hk, T, D, pairs):
    q, k = _rand((B, Hq, T, D), t, 1, 1.5), _rand((B, Hk, T, D), t, 2)
    w = [_rand((D,), t, 3 + i, 0.2, 1.0) for i in range(2)] if norm else [None, None]
    positions = torch.arange(T, device="cuda")[None] + 1000 * torch.arange(B, device="cuda")[:, None]
    _check(q, k, *w, positions.int(), _frequencies(pairs), interleaved, norm=norm)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D", [2, 3, 5, 8, 9, 15, 17, 24, 31, 33, 47, 63, 75, 100, 129, 253])
def test_every_end_of_a_row(gpu, t, interleaved, D):
    # pairs and what is not rotated end anywhere inside an item
    at, w = torch.arange(3, device="cuda"), _rand((D,), t, 3)
    for pairs in sorted({1, 2, 3, 4, 5, 8, 9, D // 4, D // 2 - 1, D // 2}):
        if 1 <= pairs <= D // 2:
            q, k = _rand((1, 3, 3, D), t, pairs), _rand((1, 1, 3, D), t, 2)
            _check(q, k, w, w, at, _frequencies(pairs), interleaved)
            _check(q, k, None, None, at, _frequencies(pairs), interleaved, norm=False)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("norm", [False, True])
def test_axes_and_shared_positions(gpu, t, norm):
    B, T, D = 2, 50, 64
    q, k = _rand((B, 4, T, D), t, 1), _rand((B, 2, T, D), t, 2)
    w = [_rand((D,), torch.float32, 3 + i) for i in range(2)] if norm else [None, None]
    at = torch.arange(T, device="cuda")
    grid = torch.stack([at // 7, at % 7], -1)
    for positions, f in ((grid.int(), _frequencies(16, 2)), (grid[None].expand(B, T, 2), _frequencies(16, 2)),
                         (torch.stack([at, at // 7, at % 7], -1).int(), _frequencies(8, 3)),
                         (at, _frequencies(32)), (at.int()[None].expand(B, T), _frequencies(32)),
                         (torch.stack([at, at, at], 0)[:2, :].int()[:, ::1], _frequencies(3))):
        _check(q, k, *w, positions, f, norm=norm)


def test_far_and_negative_positions(gpu):
    # a float32 angle would be off by 64 at 2^30; the phase is an integer and is not
    q = _rand((1, 2, 6, 64), torch.float32, 1)
    p32 = torch.tensor([2 ** 31 - 1, -2 ** 31, 2 ** 30 + 1, -1, 0, 123456789], device="cuda", dtype=torch.int32)
    p64 = torch.tensor([2 ** 40 + 7, -2 ** 62, 2 ** 63 - 1, -1, 0, 2 ** 33], device="cuda")
    for p in (p32, p64):
        _check(q, None, None, None, p, _frequencies(32), norm=False)
        _check(q, None, None, None, p, _frequencies(32), norm=True)
    # and against the angle itself, as far as float64 has it
    from blitzgs_amd.rotary import rotate
    x = torch.zeros((1, 1, 2, 64), device="cuda")
    x[..., :32] = 1.0
    at = torch.tensor([2 ** 31 - 1, 1], device="cuda")
    y = rotate(x, None, at, _frequencies(32))[0].double().cpu()[0, 0]
    angle = at.cpu().double()[:, None] * torch.tensor([10000.0 ** (-i / 32) for i in range(32)], dtype=torch.float64)
    # float64 angles of 2^31 are off by 2^-22, frequencies by a 2^-53rd of them twice
    assert (y[:, :32] - torch.cos(angle)).abs().max() < 2e-6 and (y[:, 32:] - torch.sin(angle)).abs().max() < 2e-6


@pytest.mark.parametrize("t", TYPES)
def test_strides_and_magnitude(gpu, t):
    B, T, D = 2, 21, 48
    fused = _rand((B, T, 9, D), t, 1)                          # a fused projection's slices
    q, k = fused[:, :, :4].transpose(1, 2), fused[:, :, 4:6].transpose(1, 2)
    f, at = _frequencies(12), torch.arange(100, 100 + T, device="cuda").int()
    w = _rand((2 * D,), t, 2)[1::2]                            # not contiguous
    _check(q, k, w, None, at, f, magnitude=1.25)
    _check(q, k, None, None, at, f, magnitude=-0.5, norm=False)
    odd = _rand((B, 3, T, D + 1), t, 3)[..., 1:]               # rows that start off 16 bytes
    _check(odd, k, None, w.float(), at, f)
    _check(_rand((B, 3, D, T), t, 4).transpose(2, 3), None, None, None, at, f, True)   # the last dimension not contiguous
    _check(_rand((B, 1, T, D), t, 5).expand(B, 4, T, D), None, w, None, at, f)         # one head for all
    spread = torch.stack([at, at], -1)[:, 0]                   # positions apart
    _check(q, k, None, None, spread, f, norm=False)


def test_weights_alone_and_one_side(gpu):
    from blitzgs_amd.rotary import norm_rotate
    t = torch.bfloat16
    q, k = _rand((1, 2, 5, 16), t, 1), _rand((1, 1, 5, 16), t, 2)
    f, at = _frequencies(8), torch.arange(5, device="cuda")
    w = _rand((16,), t, 3).requires_grad_(True)
    a = norm_rotate(q, k, w, None, at, f)
    (g,) = torch.autograd.grad(a, w, [torch.ones_like(x) for x in a])
    want = rotary_64(q, w, torch.ones_like(a[0]), at, f, False, 1.0, True, 1e-6)
    within(g, *want["dw"], "dw")
    # only k's rows are asked for, and only q's result is used
    kl = k.clone().requires_grad_(True)
    a = norm_rotate(q, kl, None, None, at, f)
    (g,) = torch.autograd.grad(a[0].sum() * 0 + a[1].float().sum(), kl)
    within(g, *rotary_64(k, None, torch.ones_like(k), at, f, False, 1.0, True, 1e-6)["dx"], "dk")


def test_nothing_and_nan(gpu):
    from blitzgs_amd.rotary import norm_rotate, rotate
    f = _frequencies(8)
    for shape in ((0, 2, 3, 16), (2, 2, 0, 16), (2, 0, 3, 16)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        w = torch.ones(16, device="cuda", requires_grad=True)
        y = norm_rotate(x, None, w, None, torch.zeros(shape[2], device="cuda", dtype=torch.int32), f)[0]
        assert y.shape == shape
        y.sum().backward()
        assert torch.equal(w.grad, torch.zeros_like(w)) and x.grad.shape == shape
    x = _rand((1, 2, 4, 16), torch.float32, 1)
    at = torch.arange(4, device="cuda")
    clean = rotate(x, None, at, f)[0]
    x[0, 1, 2, 3] = float("nan")
    y = rotate(x, None, at, f)[0]
    bad = torch.isnan(y)
    assert bad[0, 1, 2, 3] and bad[0, 1, 2, 11] and bad.sum() == 2 and torch.equal(y[~bad], clean[~bad])
    z = norm_rotate(torch.zeros_like(x), None, None, None, at, f)[0]
    assert torch.equal(z, torch.zeros_like(z))


def test_a_weight_of_no_heads(gpu):
    # its gradient is zero, also where the other side asks for none
    from blitzgs_amd.rotary import norm_rotate
    at, f = torch.arange(5, device="cuda"), _frequencies(4)
    for k in (None, torch.ones((2, 3, 5, 16), device="cuda")):
        w = torch.ones(16, device="cuda", requires_grad=True)
        y, _ = norm_rotate(torch.ones((2, 0, 5, 16), device="cuda"), k, w, None, at, f)
        torch.full((16,), math.nan, device="cuda")      # what a gradient that is not written may hold
        (g,) = torch.autograd.grad(y, w, torch.ones_like(y))
        assert torch.equal(g, torch.zeros_like(w))


def test_gradient_against_differences(gpu):
    # f = sum(y c): central differences along a random direction in fp32 with steps of 1e-2, as for layer norm
    from blitzgs_amd.rotary import norm_rotate
    f, at = _frequencies(5), torch.arange(6, device="cuda")
    args = [_rand((2, 3, 6, 24), torch.float32, 0), _rand((2, 1, 6, 24), torch.float32, 1),
            _rand((24,), torch.float32, 2), _rand((24,), torch.float32, 3)]
    c = [_rand(x.shape, torch.float32, 8) for x in args[:2]]
    value = lambda *a: sum((y.double() * d.double()).sum().item()  # noqa: E731
                           for y, d in zip(norm_rotate(*a, at, f), c))
    leaves = [a.clone().requires_grad_(True) for a in args]
    grads = torch.autograd.grad(norm_rotate(*leaves, at, f), leaves, c)
    for i in range(4):
        d = _rand(args[i].shape, torch.float32, 20 + i)
        d /= d.norm()
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + 1e-2 * d, args[i] - 1e-2 * d
        along = (grads[i].double() * d.double()).sum().item()
        assert abs((value(*up) - value(*down)) / 2e-2 - along) <= 1e-2 * (1 + abs(along))


def test_frequencies(gpu):
    from blitzgs_amd.rotary import as_turns, rotary_frequencies
    turns = lambda f: f.double().cpu() / 2.0 ** 64 * 2 * math.pi  # noqa: E731
    plain = torch.tensor([10000.0 ** (-i / 16) for i in range(16)], dtype=torch.float64)
    assert torch.allclose(turns(rotary_frequencies(16)), plain, rtol=1e-14, atol=0)
    assert torch.allclose(turns(rotary_frequencies(16, factor=4.0)), plain / 4, rtol=1e-14, atol=0)
    part = turns(rotary_frequencies(16, factor=4.0, trained=2048, ramp=(1.0, 32.0)))
    count = plain * 2048 / (2 * math.pi)
    assert torch.allclose(part[count >= 32], plain[count >= 32]) and torch.allclose(part[count <= 1], plain[count <= 1] / 4)
    mid = (count > 1) & (count < 32)
    kept = (count - 1) / 31
    assert mid.any() and torch.allclose(part[mid], (plain * (kept + (1 - kept) / 4))[mid])
    assert rotary_frequencies(4, axes=3).shape == (3, 4)
    # whole turns do not count, half a turn and negative angles are held
    f = as_turns([2 * math.pi, math.pi, -1.0, 7.0], device="cuda")
    assert f.tolist()[:2] == [0, -2 ** 63] and abs(turns(f)[2] + 1) < 1e-14 and abs(turns(f)[3] - (7 - 2 * math.pi)) < 1e-14
    for bad in (dict(pairs=0), dict(pairs=4, base=0.0), dict(pairs=4, factor=math.inf), dict(pairs=4, trained=0),
                dict(pairs=4, trained=5, ramp=(3.0, 3.0))):
        with pytest.raises(RuntimeError):
            rotary_frequencies(**bad)
    with pytest.raises(RuntimeError):
        as_turns([math.nan])


def test_equal_bits_and_another_stream(gpu):
    from blitzgs_amd.rotary import norm_rotate
    q, k = _rand((2, 8, 3000, 64), torch.bfloat16, 1), _rand((2, 2, 3000, 64), torch.bfloat16, 2)
    w, f, at = _rand((64,), torch.float32, 3), _frequencies(32), torch.arange(3000, device="cuda")

    def once():
        leaves = [x.clone().requires_grad_(True) for x in (q, k, w)]
        y = norm_rotate(leaves[0], leaves[1], leaves[2], leaves[2], at, f)
        return [x.detach() for x in y] + list(torch.autograd.grad(y, leaves, (q, k)))

    first = once()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = once()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_refusals(gpu):
    from blitzgs_amd.rotary import norm_rotate, rotate
    q, k = torch.zeros((2, 4, 3, 16), device="cuda"), torch.zeros((2, 2, 3, 16), device="cuda")
    at, f, w = torch.arange(3, device="cuda"), _frequencies(8), torch.ones(16, device="cuda")
    good = [q, k, w, w, at, f]
    norm_rotate(*good)
    for i, bad, words in [
            (0, q.cpu(), "HIP device tensor"), (0, q.double(), "float32, bfloat16 or float16"), (0, q[0], "dimensions"),
            (0, torch.zeros((2, 4, 3, 257), device="cuda"), "dimensions"), (1, k.bfloat16(), "k must have"),
            (1, k[:, :, :2], "k must have"), (1, k[:1], "k must have"), (2, w[:8], "q_weight"), (3, w.half(), "k_weight"),
            (4, at.float(), "positions"), (4, at[:2], "positions"), (4, at.cpu(), "positions"),
            (4, at[None].expand(3, 3), "positions"), (4, at[:, None], "positions"), (5, f.int(), "frequencies"),
            (5, _frequencies(9), "frequencies"), (5, f.cpu(), "frequencies"), (5, f[:0], "frequencies"),
            (5, f.view(1, 2, 4), "frequencies")]:
        args = list(good)
        args[i] = bad
        with pytest.raises(RuntimeError, match=words):
            norm_rotate(*args)
    with pytest.raises(RuntimeError, match="below 2\\^31"):
        rotate(q[:, :1].expand(2, 1 << 31, 3, 16), None, at, f)
    with pytest.raises(RuntimeError, match="k_weight needs k"):
        norm_rotate(q, None, None, w, at, f)
    with pytest.raises(RuntimeError, match="one type"):
        norm_rotate(q.bfloat16(), k.bfloat16(), w, w.bfloat16(), at, f)
    for m in (math.nan, math.inf, 1e39):
        with pytest.raises(RuntimeError, match="magnitude"):
            rotate(q, k, at, f, magnitude=m)
    with pytest.raises(RuntimeError, match="eps"):
        norm_rotate(*good, eps=-1.0)
