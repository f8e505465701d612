"""A block of a token network as it is trained and used: layer norm, a fused projection,
norm_rotate, attention, feed_forward and the updates of AdamW and OrthogonalMomentum
together; the operators in captured graphs, behind hooks on saved tensors and in
checkpoints; what autograd is told; kernels in the timing."""
import math

import pytest
import torch
from torch import nn

from token_helpers import TYPES

pytestmark = pytest.mark.gpu


def _rand(shape, seed, t=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(t)


B, T, W, HEADS, KEYS, D, H = 2, 37, 96, 4, 2, 24, 160
SHAPES = dict(norm1=(W,), norm2=(W,), qw=(D,), kw=(D,), qkv=((HEADS + 2 * KEYS) * D, W), proj=(W, HEADS * D),
              gate=(H, W), up=(H, W), down=(W, H))


def _params(t, device="cuda"):
    return {k: ((_rand(s, i) / math.sqrt(s[-1])) if len(s) == 2 else 1 + 0.1 * _rand(s, i)).to(t).to(device)
            for i, (k, s) in enumerate(SHAPES.items())}


def _angles():
    from blitzgs_amd.rotary import rotary_frequencies
    at = torch.arange(T, device="cuda")
    return torch.stack([at // 7, at % 7], -1), rotary_frequencies(6, axes=2)


def _block(x, p, positions, frequencies, lengths):
    from blitzgs_amd.attention import attention
    from blitzgs_amd.feedforward import feed_forward
    from blitzgs_amd.norm import layer_norm
    from blitzgs_amd.rotary import norm_rotate
    t = x.dtype
    qkv = (layer_norm(x, p["norm1"]) @ p["qkv"].t().to(t)).view(B, T, -1, D)
    q, k, v = (s.transpose(1, 2) for s in qkv.split([HEADS, KEYS, KEYS], 2))
    q, k = norm_rotate(q, k, p["qw"], p["kw"], positions, frequencies)
    o = attention(q, k, v, key_lengths=lengths).transpose(1, 2).reshape(B, T, -1)
    x = x + o @ p["proj"].t().to(t)
    return x + feed_forward(layer_norm(x, p["norm2"]), *(p[n].to(t) for n in ("gate", "up", "down")))


def _block_64(x, p, positions, frequencies, lengths):
    def norm(x, w):
        return nn.functional.layer_norm(x, (W,)) * w

    def rotate(x, w):
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
        angle = (positions[..., None].cpu() * frequencies.cpu()).flatten(1).double() * (2 * math.pi / 2.0 ** 64)
        N = angle.shape[-1]
        a, b = x[..., :N], x[..., N:2 * N]
        c, s = torch.cos(angle), torch.sin(angle)
        return torch.cat([a * c - b * s, a * s + b * c, x[..., 2 * N:]], -1)

    qkv = (norm(x, p["norm1"]) @ p["qkv"].T).view(B, T, -1, D)
    q, k, v = (s.transpose(1, 2) for s in qkv.split([HEADS, KEYS, KEYS], 2))
    q, k = rotate(q, p["qw"]), rotate(k, p["kw"])
    k, v = (s.repeat_interleave(HEADS // KEYS, 1) for s in (k, v))
    S = q @ k.transpose(2, 3) / math.sqrt(D)
    S = S.masked_fill(torch.arange(T) >= lengths.cpu().view(B, 1, 1, 1), -math.inf)
    o = (torch.softmax(S, -1) @ v).transpose(1, 2).reshape(B, T, -1)
    x = x + o @ p["proj"].T
    h = norm(x, p["norm2"])
    return x + (nn.functional.silu(h @ p["gate"].T) * (h @ p["up"].T)) @ p["down"].T


@pytest.mark.parametrize("t", TYPES)
def test_a_block_and_its_gradients(gpu, t):
    # about 20 roundings of relative size u lie between the inputs and a gradient, each of which the block
    # passes on with a factor near one; in fp32 sums of up to 160 terms add their own
    from token_helpers import U
    positions, frequencies = _angles()
    lengths = torch.tensor([T, 11], device="cuda", dtype=torch.int32)
    p = {k: v.requires_grad_(True) for k, v in _params(t).items()}
    x, dy = _rand((B, T, W), 90, t).requires_grad_(True), _rand((B, T, W), 91, t)
    y = _block(x, p, positions, frequencies, lengths)
    got = [y.detach(), *torch.autograd.grad(y, [x, *p.values()], dy)]
    p64 = {k: v.detach().double().cpu().requires_grad_(True) for k, v in p.items()}
    x64 = x.detach().double().cpu().requires_grad_(True)
    y64 = _block_64(x64, p64, positions, frequencies, lengths)
    want = [y64.detach(), *torch.autograd.grad(y64, [x64, *p64.values()], dy.double().cpu())]
    for name, a, b in zip(["y", "dx", *p], got, want):
        rel = ((a.double().cpu() - b).norm() / b.norm()).item()
        assert rel <= 20 * (U[t] + 160 ** 0.5 * U[torch.float32]), (name, rel)


def test_a_block_is_trained(gpu):
    # both optimisers on one network: the state they keep, and parameters that all move
    from blitzgs_amd.adamw import AdamW
    from blitzgs_amd.orthogonal import OrthogonalMomentum
    positions, frequencies = _angles()
    lengths = torch.tensor([T, 11], device="cuda", dtype=torch.int32)
    for bits in (32, 8):
        p = {k: nn.Parameter(v) for k, v in _params(torch.float32).items()}
        opt = [OrthogonalMomentum([v for v in p.values() if v.dim() == 2], lr=0.01),
               AdamW([v for v in p.values() if v.dim() == 1], lr=1e-2, bits=bits)]
        before = {k: v.detach().clone() for k, v in p.items()}
        x = _rand((B, T, W), 90, torch.bfloat16)
        for _ in range(3):
            for o in opt:
                o.zero_grad(set_to_none=True)
            _block(x, p, positions, frequencies, lengths).float().square().mean().backward()
            for o in opt:
                o.step()
        assert all(torch.isfinite(v).all() and not torch.equal(v, before[k]) for k, v in p.items())


def test_one_token_at_a_time(gpu):
    # a sequence's last token alone gives what the whole sequence gives there: its rotation by its own position
    from blitzgs_amd.rotary import norm_rotate, rotary_frequencies
    f, at = rotary_frequencies(12), torch.arange(1000, 1000 + T, device="cuda")
    for t in TYPES:
        q, k, w = _rand((B, HEADS, T, D), 1, t), _rand((B, KEYS, T, D), 2, t), _rand((D,), 3, t)
        every = norm_rotate(q, k, w, w, at, f)
        for i in (0, 17, T - 1):
            one = norm_rotate(q[:, :, i:i + 1], k[:, :, i:i + 1], w, w, at[i:i + 1], f)
            assert all(torch.equal(a, b[:, :, i:i + 1]) for a, b in zip(one, every))


def _replays(make, change, times=4):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        make()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = make()
    for i in range(times):
        change(i)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(kept, make()):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("norm", [False, True])
def test_rotation_in_a_graph(gpu, norm):
    from blitzgs_amd.rotary import norm_rotate, rotary_frequencies, rotate
    q, k = _rand((2, 4, 300, 64), 0).requires_grad_(True), _rand((2, 2, 300, 64), 1).requires_grad_(True)
    w = _rand((64,), 2).requires_grad_(True)
    f, at = rotary_frequencies(16), torch.arange(300, device="cuda")

    def make():
        y = norm_rotate(q, k, w, w, at, f) if norm else rotate(q, k, at, f)
        leaves = (q, k, w) if norm else (q, k)
        return [*(a.detach() for a in y), *torch.autograd.grad(y, leaves, [torch.ones_like(a) for a in y])]

    def change(i):
        q.data.copy_(_rand(q.shape, 10 + i))
        at.add_(1000 * i)

    _replays(make, change)


# large, split, odd, single-row and large odd shapes
@pytest.mark.parametrize("M,W,H,t", [(2100, 264, 520, torch.bfloat16), (700, 64, 128, torch.float32),
                                     (90, 33, 65, torch.float16), (1, 512, 1024, torch.bfloat16),
                                     (8, 512, 1030, torch.float32), (800, 515, 1001, torch.bfloat16)])
def test_feed_forward_in_a_graph(gpu, M, W, H, t):
    from blitzgs_amd.feedforward import feed_forward
    leaves = [_rand(s, i, t, s[-1] ** -0.5 if i else 1.0).requires_grad_(True)
              for i, s in enumerate([(M, W), (H, W), (H, W), (W, H)])]
    dy = _rand((M, W), 9, t)

    def make():
        y = feed_forward(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    _replays(make, lambda i: leaves[0].data.copy_(_rand((M, W), 10 + i, t)))


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_update_in_a_graph(gpu, bits):
    from blitzgs_amd.adamw import adamw_update, new_moments
    sizes = [300, 5000]
    p, g = [_rand((n,), n) for n in sizes], [_rand((n,), n + 1) for n in sizes]
    m, v, s = (list(x) for x in zip(*[new_moments(x, bits) for x in p]))
    state = [*p, *m, *v, *(s if bits == 8 else [])]
    kept = [torch.empty_like(x) for x in state]
    start = [x.clone() for x in state]

    def make():
        for x, y in zip(state, start):
            x.copy_(y)
        adamw_update(p, g, m, v, step=3, lr=0.1, scales=s if bits == 8 else None)
        for x, y in zip(kept, state):
            x.copy_(y)
        return [x.clone() for x in kept]

    _replays(make, lambda i: g[0].copy_(_rand((300,), 20 + i)))


def test_two_graphs_and_eager_calls_between(gpu):
    # two captured calls have workspaces of their own
    from blitzgs_amd.feedforward import feed_forward
    made = []
    for seed in (0, 50):
        leaves = [_rand(s, seed + i).requires_grad_(True) for i, s in enumerate([(60, 256), (512, 256), (512, 256), (64, 512)])]
        call = lambda leaves=leaves: [(y := feed_forward(*leaves)).detach(),  # noqa: E731
                                      *torch.autograd.grad(y, leaves, torch.ones_like(y))]
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            call()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        made.append((graph, out, call))
    for _ in range(3):
        for graph, _, _ in made:
            graph.replay()
        want = [call() for _, _, call in made]
        torch.cuda.synchronize()
        for (_, out, _), w in zip(made, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w))


def _packed(t):
    return torch.empty(t.size(), device=t.device, dtype=t.dtype).copy_(t)


def _turned(t):
    return _packed(t.permute(*reversed(range(t.dim())))).permute(*reversed(range(t.dim())))


def _spread(t):
    return torch.empty((*t.shape, 2), device=t.device, dtype=t.dtype)[..., 0].copy_(t)


def _off(t):
    # bytes from an odd address on
    return torch.empty(t.numel() + 1, device=t.device, dtype=t.dtype)[1:].copy_(t) if t.dtype == torch.uint8 else t


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("kind", ["cpu", "packed", "turned", "spread", "off"])
def test_saved_tensors_in_other_places(gpu, kind, t):
    from blitzgs_amd.feedforward import feed_forward
    from blitzgs_amd.rotary import norm_rotate, rotary_frequencies
    fused, w = _rand((B, T, HEADS + 2 * KEYS, D), 1, t), _rand((D,), 2, t)
    at = torch.stack([torch.arange(T, device="cuda")] * 2)
    f = rotary_frequencies(6)

    def grads():
        leaf, wl = fused.clone().requires_grad_(True), w.clone().requires_grad_(True)
        q, k = leaf[:, :, :HEADS].transpose(1, 2), leaf[:, :, HEADS:HEADS + KEYS].transpose(1, 2)
        a = norm_rotate(q, k, wl, wl, at, f)
        x = _rand((50, 3 * 40), 3, t)[:, 40:80].requires_grad_(True)
        leaves = [_rand(s, 4 + i, t, 0.2).requires_grad_(True) for i, s in enumerate([(72, 40), (72, 40), (24, 72)])]
        y = feed_forward(x, *leaves)
        outs = [*a, y]
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, [leaf, wl, x, *leaves],
                                                                     [torch.ones_like(o) for o in outs]))

    want = grads()
    through = torch.autograd.graph.save_on_cpu() if kind == "cpu" else torch.autograd.graph.saved_tensors_hooks(
        dict(packed=_packed, turned=_turned, spread=_spread, off=_off)[kind], lambda t: t)
    with through:
        got = grads()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_checkpointed_blocks(gpu):
    from torch.utils.checkpoint import checkpoint
    positions, frequencies = _angles()
    lengths = torch.tensor([T, 11], device="cuda", dtype=torch.int32)
    p = {k: v.requires_grad_(True) for k, v in _params(torch.bfloat16).items()}

    def grads(run):
        leaf = _rand((B, T, W), 90, torch.bfloat16).requires_grad_(True)
        y = run(lambda a: _block(a, p, positions, frequencies, lengths), leaf)
        return torch.autograd.grad(y, [leaf, *p.values()], torch.ones_like(y))

    want = grads(lambda f, a: f(a))
    got = grads(lambda f, a: checkpoint(f, a, use_reentrant=False))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_forward_mode_and_second_derivatives_are_refused(gpu):
    from torch.autograd import forward_ad

    from blitzgs_amd.feedforward import feed_forward
    from blitzgs_amd.rotary import rotary_frequencies, rotate
    q, f, at = _rand((1, 2, 3, 8), 0), rotary_frequencies(4), torch.arange(3, device="cuda")
    x, ws = _rand((4, 8), 1), [_rand((8, 8), i) for i in (2, 3, 4)]
    with forward_ad.dual_level():
        dual = lambda a: forward_ad.make_dual(a, torch.ones_like(a))  # noqa: E731
        with pytest.raises(NotImplementedError, match="jvp|forward"):
            rotate(dual(q), None, at, f)
        with pytest.raises(NotImplementedError, match="jvp|forward"):
            feed_forward(x, ws[0], dual(ws[1]), ws[2])
    leaf = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(feed_forward(leaf, *ws).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), leaf)


def test_the_kernels_are_timed(gpu):
    from blitzgs_amd import _lib
    from blitzgs_amd.adamw import AdamW
    positions, frequencies = _angles()
    p = {k: nn.Parameter(v) for k, v in _params(torch.float32).items()}
    opt = AdamW(p.values(), bits=8)
    _lib.timing_reset()
    _lib.timing_enable(True)
    try:
        _block(_rand((B, T, W), 90), p, positions, frequencies, None).sum().backward()
        opt.step()
        torch.cuda.synchronize()
        names = set(_lib.timing_read())
    finally:
        _lib.timing_enable(False)
        _lib.timing_reset()
    assert {"rotary_fwd_kernel", "rotary_bwd_kernel", "rotary_columns_kernel", "feed_small_kernel", "adamw_kernel"} <= names
