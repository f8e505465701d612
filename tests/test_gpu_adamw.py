"""adamw_update and AdamW against their 64-bit forms: types, sizes about blocks of 128
and chunks, more tensors than one launch takes, odd addresses; 8-bit moments code by
code, their mean over many steps, NaN and infinities; the optimiser's state."""
import copy
import math

import pytest
import torch

from block_helpers import adamw_64, codes_8, draws, values_8
from token_helpers import TYPES, within

pytestmark = pytest.mark.gpu
HOW = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
SIZES = [1, 7, 8, 127, 128, 129, 1000, 2047, 2048, 2049, 5000]


def _rand(shape, t, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(t)


def _apart(sizes, t, seed, scale=1.0):
    """Tensors of one buffer, at odd places."""
    buffer, at, out = _rand((sum(sizes) + 3 * len(sizes) + 1,), t, seed, scale), 1, []
    for n in sizes:
        out.append(buffer[at:at + n])
        at += n + 3
    return buffer, out


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("step", [1, 2, 1000])
def test_moments_in_32_bits(gpu, t, step):
    from blitzgs_amd.adamw import adamw_update
    (pb, p), (gb, g) = _apart(SIZES, t, 1), _apart(SIZES, t, 2, 0.1)
    (mb, m), (vb, v) = _apart(SIZES, torch.float32, 3, 0.01), _apart(SIZES, torch.float32, 4, 0.01)
    vb.square_()
    before = [x.clone() for x in (pb, gb, mb, vb)]
    keep = [[x.clone() for x in xs] for xs in (p, g, m, v)]
    adamw_update(p, g, m, v, step=step, **HOW)
    for i in range(len(SIZES)):
        p0, g0, m0, v0 = (k[i] for k in keep)
        want = adamw_64(p0, g0, m0.double().cpu(), v0.double().cpu(), step, HOW["lr"], HOW["betas"], HOW["eps"],
                        HOW["weight_decay"])
        for got, w, name in zip((p[i], m[i], v[i]), want, "pmv"):
            within(got, *w, f"{name} of {SIZES[i]}")
    # what lies between the tensors is as it was, and the gradients
    for buffer, old, tensors in ((pb, before[0], p), (mb, before[2], m), (vb, before[3], v)):
        inside = torch.zeros_like(buffer, dtype=torch.bool)
        for x in tensors:
            inside[x.storage_offset():x.storage_offset() + x.numel()] = True
        assert torch.equal(buffer[~inside], old[~inside])
    assert torch.equal(gb, before[1])


def _packed(sizes, seed):
    """8-bit moments as some earlier step left them: any codes but NaN's."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ints = lambda n, top: torch.randint(0, top, (n,), generator=g, device="cuda")  # noqa: E731
    m = [(ints(n, 121) + 128 * ints(n, 2)).to(torch.uint8) for n in sizes]
    v = [ints(n, 249).to(torch.uint8) for n in sizes]
    s = [torch.stack([110 + ints(-(-n // 128), 5), 95 + ints(-(-n // 128), 5)]).to(torch.uint8) for n in sizes]
    return m, v, s


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("step,seed", [(1, 0), (77, 123), (2 ** 40 + 3, -5)])
def test_moments_in_8_bits(gpu, t, step, seed):
    from blitzgs_amd.adamw import adamw_update, moment_values
    p, g = _apart(SIZES, t, 1)[1], _apart(SIZES, t, 2, 1e-4)[1]
    m, v, s = _packed(SIZES, 3)
    keep = [[x.clone() for x in xs] for xs in (p, g, m, v, s)]
    adamw_update(p, g, m, v, step=step, scales=s, seed=seed, **HOW)
    for i, n in enumerate(SIZES):
        p0, g0, m0, v0, s0 = (k[i] for k in keep)
        want = adamw_64(p0, g0, values_8(m0, s0[0], 14), values_8(v0, s0[1], 30), step, HOW["lr"], HOW["betas"],
                        HOW["eps"], HOW["weight_decay"])
        within(p[i], *want[0], f"p of {n}")
        bits = draws(n, i, step, seed & 0xFFFFFFFF)
        for got, scales, (x, e), draw, top in ((m[i], s[i][0], want[1], bits & 65535, 14),
                                               (v[i], s[i][1], want[2], bits >> 16, 30)):
            low, high, unit = codes_8(x, draw, top, e)
            c = got.cpu().long()
            size = c & 127 if top == 14 else c
            assert torch.equal(scales.cpu().long(), unit.long()), (n, top)
            assert ((low <= size) & (size <= high)).all(), (n, top)
            # the bounds are the same code but where the rest is at a border
            assert (low == high).double().mean() > 0.99
            if top == 14:
                assert torch.equal((c >= 128)[size > 0], (x < 0)[size > 0])
        for dtype in (torch.float32, torch.bfloat16):
            a, b = moment_values(m[i], v[i], s[i], dtype=dtype)
            assert torch.equal(a.double().cpu(), values_8(m[i], s[i][0], 14))
            assert torch.equal(b.double().cpu(), values_8(v[i], s[i][1], 30))


def test_more_tensors_than_a_launch_and_large_ones(gpu):
    from blitzgs_amd.adamw import adamw_update, new_moments
    sizes = [(i * 37) % 300 for i in range(130)] + [70001]         # empty ones among them
    for bits in (32, 8):
        p, g = [_rand((n,), torch.float32, n) for n in sizes], [_rand((n,), torch.float32, n + 1) for n in sizes]
        one = [x.clone() for x in p]
        moments = [new_moments(x, bits) for x in p]
        adamw_update(p, g, *zip(*[x[:2] for x in moments]), step=3, scales=[x[2] for x in moments] if bits == 8 else None,
                     **HOW)
        for x, y, q in zip(p, one, g):
            want = adamw_64(y, q, torch.zeros(x.shape, dtype=torch.float64), torch.zeros(x.shape, dtype=torch.float64), 3,
                            HOW["lr"], HOW["betas"], HOW["eps"], HOW["weight_decay"])
            within(x, *want[0], str(x.numel()))


def test_rounding_keeps_the_mean(gpu):
    # no gradient: v falls by a thousandth a step, far below the distance of two codes.  Of n = 2^16 equal
    # elements each step's rounding leaves the mean where it is: after k steps the mean is 0.999^k of the
    # start's, with a variance of at most k (step / 2)^2 / n: step is at most 1/8 of the value
    from blitzgs_amd.adamw import adamw_update, moment_values, new_moments
    n, k = 1 << 16, 200
    p = torch.zeros(n, device="cuda")
    g = torch.zeros(n, device="cuda")
    m, v, s = new_moments(p, 8)
    start = torch.full((n,), 1.0, device="cuda")
    start[::128] = 1.9                                             # keeps the blocks' powers of two
    adamw_update([p], [start], [m], [v], step=1, lr=0.0, betas=(0.5, 0.999), scales=[s])
    v0 = moment_values(m, v, s)[1].double()
    for i in range(k):
        adamw_update([p], [g], [m], [v], step=2 + i, lr=0.0, betas=(0.5, 0.999), scales=[s])
    m1, v1 = moment_values(m, v, s)
    few = slice(1, 128)
    ratio = (v1.double().view(-1, 128)[:, few].mean() / v0.view(-1, 128)[:, few].mean()).item()
    noise = math.sqrt(k) * (1 / 16) / math.sqrt(n)
    assert abs(ratio - 0.999 ** k) <= 6 * noise and ratio < 0.9
    assert not torch.equal(v1, v0.float())


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-12])
def test_small_gradients_and_a_small_eps(gpu, bits, eps):
    # second moments below fp32's normal range, which eps does not hide
    from blitzgs_amd.adamw import adamw_update, new_moments
    p = _rand((500,), torch.float32, 1)
    g = _rand((500,), torch.float32, 2).sign() * torch.logspace(-20, -15, 500, device="cuda")
    q = p.clone()
    m, v, s = new_moments(q, bits)
    how = dict(lr=0.1, betas=(0.9, 0.999), eps=eps, weight_decay=0.0)
    adamw_update([q], [g], [m], [v], step=1, scales=None if bits == 32 else [s], **how)
    g64 = g.double()
    want = p.double() - 0.1 * g64 / (g64.abs() + eps)
    # a subnormal v has a last bit of 2^-149: its root is off by that over twice the root; the update is at most 0.1
    loose = 0.1 * torch.clamp(2.0 ** -149 / (0.001 * g64.square()), max=2.0) + 20 * 2.0 ** -24
    assert ((q.double() - want).abs() <= loose + 2.0 ** -24 * p.abs().double()).all()


def test_zero_nan_and_infinity(gpu):
    from blitzgs_amd.adamw import adamw_update, moment_values, new_moments
    n = 300
    p, g = _rand((n,), torch.float32, 1), _rand((n,), torch.float32, 2)
    g[130:260] = 0.0
    g[5], g[140] = math.nan, math.inf
    clean = g.clone()
    clean[5] = clean[140] = 0.0
    out = []
    for grad in (g, clean):
        q = p.clone()
        m, v, s = new_moments(q, 8)
        adamw_update([q], [grad], [m], [v], step=1, scales=[s], **HOW)
        out.append((q, *moment_values(m, v, s), m.clone(), v.clone()))
    bad = torch.zeros(n, dtype=torch.bool, device="cuda")
    bad[5] = bad[140] = True
    for a, b in zip(out[0][:3], out[1][:3]):
        assert torch.isnan(a[bad]).all() and torch.equal(a[~bad], b[~bad])
    assert torch.equal(out[1][3][141:250], torch.zeros_like(out[1][3][141:250]))     # a block of zeros
    # tiny moments are subnormal or zero, never noise
    m, v, s = new_moments(p, 8)
    adamw_update([p.clone()], [torch.full_like(p, 1e-30)], [m], [v], step=1, scales=[s], **HOW)
    a, b = moment_values(m, v, s)
    assert (a >= 0.9e-31).all() and (a <= 1.2e-31).all() and torch.equal(b, torch.zeros_like(b))


def test_elements_that_pass_a_launch(gpu):
    # 2^27 elements and a few: many workgroups, one tensor
    from blitzgs_amd.adamw import adamw_update
    n = (1 << 27) + 5
    p = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    g = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    adamw_update([p], [g], [m], [v], step=1, lr=0.5, weight_decay=0.0)
    assert (p == -0.5).all() and torch.allclose(m, torch.full((), 0.1, device="cuda"))


def test_the_optimiser(gpu):
    # against torch's, in fp32: both round each operation, a few times 2^-24 a step
    from blitzgs_amd.adamw import AdamW
    shapes = [(40, 30), (30,), (7,), (), (3, 5, 4)]
    ours = [torch.nn.Parameter(_rand(s, torch.float32, i)) for i, s in enumerate(shapes)]
    theirs = [torch.nn.Parameter(p.detach().clone()) for p in ours]
    groups = lambda ps: [dict(params=ps[:2]), dict(params=ps[2:], lr=3e-3, weight_decay=0.0)]  # noqa: E731
    a, b = AdamW(groups(ours), lr=1e-3), torch.optim.AdamW(groups(theirs), lr=1e-3)
    for k in range(6):
        for i, (p, q) in enumerate(zip(ours, theirs)):
            skipped = i == 2 and k < 2                             # one parameter begins later: a step of its own
            p.grad = None if skipped else _rand(p.shape, torch.float32, 100 * k + i)
            q.grad = None if skipped else p.grad.clone()
        a.step()
        b.step()
        if k == 3:                                                 # through a saved state
            saved = copy.deepcopy(a.state_dict())
            a = AdamW(groups(ours), lr=1e-3)
            a.load_state_dict(saved)
    for p, q in zip(ours, theirs):
        assert (p - q).abs().max() <= 6 * 2e-7 * (1 + q.abs().max())
    assert a.state[ours[2]]["step"] == 4 and a.state[ours[0]]["step"] == 6


@pytest.mark.parametrize("t", TYPES)
def test_a_saved_state_of_8_bits(gpu, t):
    from blitzgs_amd.adamw import AdamW
    make = lambda: [torch.nn.Parameter(_rand((50, 9), t, 0)), torch.nn.Parameter(_rand((11,), t, 1))]  # noqa: E731

    def run(ps, opt, steps):
        for k in steps:
            for i, p in enumerate(ps):
                p.grad = _rand(p.shape, t, 10 * k + i)
            opt.step()

    one = make()
    opt = AdamW(one, lr=1e-2, bits=8, seed=9)
    run(one, opt, range(3))
    two = [torch.nn.Parameter(p.detach().clone()) for p in one]
    other = AdamW(two, lr=1.0, bits=8)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    for p, q in zip(one, two):
        for name in ("exp_avg", "exp_avg_sq", "scales"):
            assert other.state[q][name].dtype == torch.uint8
            assert torch.equal(other.state[q][name], opt.state[p][name])
    run(one, opt, range(3, 5))
    run(two, other, range(3, 5))
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    wide = AdamW(two, lr=1.0)
    wide.load_state_dict(copy.deepcopy(opt.state_dict()))
    wide.param_groups[0]["bits"] = 32
    with pytest.raises(RuntimeError, match="32 bits"):
        wide.step()


def test_equal_bits_and_another_stream(gpu):
    from blitzgs_amd.adamw import adamw_update
    sizes = [5000, 1, 300000]
    out = []
    s = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), s):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            p, g = [_rand((n,), torch.bfloat16, 1) for n in sizes], [_rand((n,), torch.bfloat16, 2) for n in sizes]
            m, v, c = _packed(sizes, 3)
            adamw_update(p, g, m, v, step=5, scales=c, **HOW)
            out.append([*p, *m, *v, *c])
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_refusals(gpu):
    from blitzgs_amd.adamw import AdamW, adamw_update, moment_values, new_moments
    p = [torch.zeros((3, 4), device="cuda"), torch.zeros(5, device="cuda")]
    g = [torch.ones_like(x) for x in p]
    m, v, s = (list(x) for x in zip(*[new_moments(x, 32) for x in p]))
    m8, v8, s8 = (list(x) for x in zip(*[new_moments(x, 8) for x in p]))
    adamw_update([], [], [], [], 1, 0.1)
    for args, more, words in [
            ((p, g, m, v, 0, 0.1), {}, "step"), ((p, g, m, v, 1.0, 0.1), {}, "step"), ((p, g, m, v, 1, -0.1), {}, "lr"),
            ((p, g, m, v, 1, math.nan), {}, "lr"), ((p, g, m, v, 1, 0.1), dict(betas=(1.0, 0.9)), "betas"),
            ((p, g[:1], m, v, 1, 0.1), {}, "grads"), ((p, [g[0].half(), g[1]], m, v, 1, 0.1), {}, "grads"),
            ((p, [None, g[1]], m, v, 1, 0.1), {}, "grads"), ((p, g, m8, v8, 1, 0.1), {}, "exp_avgs"),
            ((p, g, m, v, 1, 0.1), dict(scales=s8), "exp_avgs"), ((p, g, m8, v8, 1, 0.1), dict(scales=s8[:1]), "scales"),
            ((p, g, m8, v8, 1, 0.1), dict(scales=[s8[0][:, :0], s8[1]]), "scales"),
            (([p[0], p[0]], [g[0], g[0]], [m[0], m[0]], [v[0], v[0]], 1, 0.1), {}, "twice"),
            (([p[0], p[0].view(-1)[7:]], [g[0], g[1]], m, v, 1, 0.1), {}, "overlap"), ((p, [p[0], g[1]], m, v, 1, 0.1), {}, "overlaps"),
            (([p[0].t(), p[1]], g, m, v, 1, 0.1), {}, "params"), (([p[0].cpu(), p[1]], g, m, v, 1, 0.1), {}, "HIP device"),
            ((p, g, [m[0].t(), m[1]], v, 1, 0.1), {}, "exp_avgs"), ((p, g, m, v, 1, 0.1), dict(seed=1.5), "seed")]:
        with pytest.raises(RuntimeError, match=words):
            adamw_update(*args, **more)
    assert all(torch.equal(x, torch.zeros_like(x)) for x in p)
    with pytest.raises(RuntimeError, match="uint8"):
        moment_values(m[0], v[0], s8[0])
    with pytest.raises(RuntimeError, match="dtype"):
        moment_values(m8[0], v8[0], s8[0], dtype=torch.float16)
    with pytest.raises(RuntimeError, match="scales"):
        moment_values(m8[0], v8[0], s8[0][:, :0])
    for bad in (dict(lr=-1.0), dict(bits=16), dict(betas=(0.9, 1.0)), dict(seed=0.5)):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(p[0])], **bad)
    q = torch.nn.Parameter(torch.zeros(4, device="cuda"))
    q.grad = torch.ones_like(q)
    opt = AdamW([q])
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()
        torch.zeros(4, device="cuda")


def test_a_step_is_seen_by_graphs_that_hold_the_parameters(gpu):
    from blitzgs_amd.adamw import AdamW
    w = _rand((6,), torch.float32, 0).requires_grad_(True)
    y = (w * w).sum()
    w.grad = torch.ones_like(w)
    AdamW([w]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
