"""What AdamW's state is after a refused step."""
import pytest
import torch

from blitzgs_amd.adamw import AdamW


def _rand(shape, t, seed, device="cpu"):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(t).to(device)


def _params(t, device="cpu"):
    return [torch.nn.Parameter(_rand(s, t, i, device)) for i, s in enumerate([(6, 5), (9,), ()])]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_a_step_refused_in_a_capture_leaves_nothing(gpu, bits):
    one, two = _params(torch.float32, "cuda"), _params(torch.float32, "cuda")
    opt, fresh = AdamW(one, bits=bits), AdamW(two, bits=bits)
    for ps in (one, two):
        for i, p in enumerate(ps):
            p.grad = _rand(p.shape, p.dtype, i, "cuda")
    torch.cuda.synchronize()
    called = []
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        for closure in (None, lambda: called.append(1)):
            with pytest.raises(RuntimeError, match="captured"):
                opt.step(closure)
        torch.zeros(4, device="cuda")
    assert len(opt.state) == 0 and not called
    opt.step()
    fresh.step()
    assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(one, two))
