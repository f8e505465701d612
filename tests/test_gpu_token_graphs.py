"""The token operators in captured graphs, forward and backward: every replay
against the same calls made directly, on inputs that change in between."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rand(shape, seed, t=torch.float32):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(t)


def _replays(make, change, times=4):
    """The graph of make() against make() itself, on inputs that change() renews."""
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


@pytest.mark.parametrize("width", [64, 1030])
def test_layer_norm_in_a_graph(gpu, width):
    from blitzgs_amd.norm import layer_norm
    x, dy = _rand((700, width), 0).requires_grad_(True), _rand((700, width), 1)
    w, b = _rand((width,), 2).requires_grad_(True), _rand((width,), 3).requires_grad_(True)

    def make():
        y = layer_norm(x, w, b)
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), dy)]

    _replays(make, lambda i: x.data.copy_(_rand(x.shape, 10 + i)))


# a split forward and split gradients; the LDS of a whole CU
@pytest.mark.parametrize("Tq,Tk,D,t", [(2, 3000, 64, torch.bfloat16), (600, 700, 128, torch.bfloat16),
                                       (3000, 40, 64, torch.float16), (90, 200, 128, torch.float32)])
def test_attention_with_its_gradients_in_a_graph(gpu, Tq, Tk, D, t):
    from blitzgs_amd.attention import attention
    q = _rand((1, 4, Tq, D), 0, t).requires_grad_(True)
    k, v = (_rand((1, 2, Tk, D), i, t).requires_grad_(True) for i in (1, 2))
    do = _rand((1, 4, Tq, D), 3, t)
    lengths = torch.tensor([Tk], dtype=torch.int32, device="cuda")

    def make():
        o = attention(q, k, v, causal=True, key_lengths=lengths)
        return [o.detach(), *torch.autograd.grad(o, (q, k, v), do)]

    def change(i):
        q.data.copy_(_rand(q.shape, 10 + i, t))
        lengths.fill_((Tk, 0, Tk // 2, 1)[i])

    _replays(make, change)


@pytest.mark.parametrize("shape", [(3, 60, 90), (130, 2100), (16, 500, 300)])
def test_orthogonalise_in_a_graph(gpu, shape):
    from blitzgs_amd.orthogonal import orthogonalise
    g = _rand(shape, 0)
    _replays(lambda: [orthogonalise(g)], lambda i: g.copy_(_rand(shape, 10 + i)))
