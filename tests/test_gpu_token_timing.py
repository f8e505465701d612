"""The library's kernel timing names every kernel of the token operators that ran."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_an_optimiser_step_is_timed_whole(gpu):
    from blitzgs_amd import _lib
    from blitzgs_amd.orthogonal import OrthogonalMomentum
    for t in (torch.float32, torch.bfloat16, torch.float16):
        p = torch.randn((40, 60), device="cuda").to(t).requires_grad_(True)
        p.grad = torch.ones_like(p)
        opt = OrthogonalMomentum([p], lr=0.1)
        _lib.timing_reset()
        _lib.timing_enable(True)
        try:
            opt.step()
            torch.cuda.synchronize()
            names = set(_lib.timing_read())
        finally:
            _lib.timing_enable(False)
            _lib.timing_reset()
        assert names == {"momentum_kernel", "orth_small_kernel", "apply_kernel"}
