"""The token operators' backward with tensors that hooks give back in other places
than the forward had them: other strides, other memory."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _packed(t):                # rows one after another
    return torch.empty(t.size(), device=t.device, dtype=t.dtype).copy_(t)


def _turned(t):                # dense, with the dimensions' order in memory turned round
    return _packed(t.permute(*reversed(range(t.dim())))).permute(*reversed(range(t.dim())))


def _spread(t):                # twice as far apart
    return torch.empty((*t.shape, 2), device=t.device, dtype=t.dtype)[..., 0].copy_(t)


def _through(kind):
    if kind == "cpu":
        return torch.autograd.graph.save_on_cpu()
    if kind == "pinned":
        return torch.autograd.graph.save_on_cpu(pin_memory=True)
    return torch.autograd.graph.saved_tensors_hooks(dict(packed=_packed, turned=_turned, spread=_spread)[kind],
                                                    lambda t: t)


KINDS = ["cpu", "pinned", "packed", "turned", "spread"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [40, 64, 33])
def test_attention(gpu, kind, t, D):
    from blitzgs_amd.attention import attention
    g = torch.Generator(device="cuda").manual_seed(5)
    B, T, H = 2, 90, 3
    lengths = torch.tensor([90, 41], dtype=torch.int32, device="cuda")

    def grads():
        fused = torch.randn((B, T, 3, H, D), generator=g.manual_seed(5), device="cuda").to(t).requires_grad_(True)
        q, k, v = (fused[:, :, i].transpose(1, 2) for i in range(3))
        o = attention(q, k, v, causal=True, key_lengths=lengths)
        (d,) = torch.autograd.grad(o, fused, torch.ones_like(o))
        return o.detach(), d

    want = grads()
    with _through(kind):
        got = grads()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("width", [64, 65])
def test_layer_norm(gpu, kind, width):
    from blitzgs_amd.norm import layer_norm
    g = torch.Generator(device="cuda").manual_seed(5)
    wide = torch.randn((50, 3 * width + 1), generator=g, device="cuda")
    w, b = (torch.randn(width, generator=g, device="cuda").requires_grad_(True) for _ in range(2))

    def grads():
        x = wide[:, width:2 * width].detach().requires_grad_(True)
        y = layer_norm(x, w, b)
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), torch.ones_like(y))]

    want = grads()
    with _through(kind):
        got = grads()
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_checkpointed_blocks(gpu):
    from torch.utils.checkpoint import checkpoint

    from blitzgs_amd.attention import attention
    from blitzgs_amd.norm import layer_norm
    x = torch.randn((2, 50, 64), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    w = torch.ones(64, device="cuda", requires_grad=True)

    def block(x):
        h = layer_norm(x, w).view(2, 50, 4, 16).transpose(1, 2)
        return attention(h, h, h, causal=True).transpose(1, 2).reshape(2, 50, 64)

    def grads(run):
        leaf = x.clone().requires_grad_(True)
        return torch.autograd.grad(run(leaf), (leaf, w), torch.ones_like(x))

    want = grads(block)
    got = grads(lambda a: checkpoint(block, a, use_reentrant=False))
    assert all(torch.equal(a, c) for a, c in zip(got, want))
