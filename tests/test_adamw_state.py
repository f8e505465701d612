"""What AdamW's state is after a refused step, and after loading a state that torch's own
optimisers saved."""
import copy

import pytest
import torch

from blitzgs_amd.adamw import AdamW

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _rand(shape, t, seed, device="cpu"):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(t).to(device)


def _params(t, device="cpu"):
    return [torch.nn.Parameter(_rand(s, t, i, device)) for i, s in enumerate([(6, 5), (9,), ()])]


def _steps(opt, ps, numbers):
    for k in numbers:
        for i, p in enumerate(ps):
            p.grad = _rand(p.shape, p.dtype, 100 * k + i, p.device)
        opt.step()


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


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("theirs", [torch.optim.AdamW, torch.optim.Adam])
def test_a_state_of_torch(theirs, bits, t):
    # its groups say nothing of bits and seeds, its moments have the parameters' type
    ps = _params(t)
    saved = theirs([dict(params=ps[:1], lr=3e-3), dict(params=ps[1:])], weight_decay=0.0)
    _steps(saved, ps[:2], range(3))                       # the third had no gradient yet
    opt = AdamW([dict(params=ps[:1]), dict(params=ps[1:], seed=4)], bits=bits, seed=9)
    opt.load_state_dict(copy.deepcopy(saved.state_dict()))
    # these moments are not of 8 bits, whatever the optimiser was made with
    assert [g["bits"] for g in opt.param_groups] == [32, 32] and [g["seed"] for g in opt.param_groups] == [9, 9]
    assert [g["lr"] for g in opt.param_groups] == [3e-3, 1e-3]
    for p in ps[:2]:
        assert opt.state[p]["step"] == 3 and isinstance(opt.state[p]["step"], int)
        for name in ("exp_avg", "exp_avg_sq"):
            got, want = opt.state[p][name], saved.state[p][name]
            assert got.dtype == torch.float32 and torch.equal(got, want.float()) and got.data_ptr() != want.data_ptr()
    assert ps[2] not in opt.state
    # without any moments the optimiser's own bits stay
    other = AdamW(ps, bits=bits, seed=9)
    other.load_state_dict(theirs(ps, weight_decay=0.0).state_dict())
    assert other.param_groups[0]["bits"] == bits


@pytest.mark.parametrize("make,words", [
    (lambda ps: torch.optim.AdamW(ps, maximize=True), "maximize"),
    (lambda ps: torch.optim.AdamW(ps, amsgrad=True), "amsgrad"),
    (lambda ps: torch.optim.Adam(ps, weight_decay=0.1), "weight_decay"),
    (lambda ps: torch.optim.SGD(ps, lr=0.1), "betas")])
def test_a_state_that_asks_for_another_step_is_refused(make, words):
    ps = _params(torch.float32)
    opt = AdamW(ps, lr=0.5)
    before = copy.deepcopy(opt.state_dict())
    with pytest.raises(ValueError, match=words):
        opt.load_state_dict(make(ps).state_dict())
    assert opt.state_dict() == before


@pytest.mark.gpu
def test_training_goes_on_from_a_state_of_torch(gpu):
    ours, theirs = _params(torch.float32, "cuda"), _params(torch.float32, "cuda")
    start = torch.optim.AdamW(ours, lr=1e-2)
    whole = torch.optim.AdamW(theirs, lr=1e-2)
    _steps(start, ours, range(3))
    _steps(whole, theirs, range(6))
    opt = AdamW(ours)
    opt.load_state_dict(start.state_dict())
    _steps(opt, ours, range(3, 6))
    # both round each operation, a few times 2^-24 a step
    for p, q in zip(ours, theirs):
        assert (p - q).abs().max() <= 6 * 2e-7 * (1 + q.abs().max())
