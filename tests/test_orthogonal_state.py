"""The state of OrthogonalMomentum: saved and loaded, it stays in 32 bits whatever
the parameters' type, and a buffer that is not the kernels' is refused before
its address is used."""
import copy

import pytest
import torch

from blitzgs_amd.orthogonal import OrthogonalMomentum

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _param(shape, t, seed, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    return torch.nn.Parameter(torch.randn(shape, generator=g).to(t).to(device))


@pytest.mark.parametrize("t", TYPES)
def test_loaded_buffers_keep_their_32_bits(t):
    params = [_param((8, 6), t, 0), _param((5, 7), t, 1), _param((3, 3), t, 2)]
    first = OrthogonalMomentum([dict(params=params[:1]), dict(params=params[1:], lr=0.2)], lr=0.1)
    for p in params[:2]:                      # the third had no gradient yet
        first.state[p]["momentum_buffer"] = torch.randn(p.shape)
    second = OrthogonalMomentum([dict(params=params[:1]), dict(params=params[1:])], lr=0.3)
    second.load_state_dict(first.state_dict())
    for p in params[:2]:
        got, want = second.state[p]["momentum_buffer"], first.state[p]["momentum_buffer"]
        assert got.dtype == torch.float32 and torch.equal(got, want)
        assert got.data_ptr() != want.data_ptr()
    assert "momentum_buffer" not in second.state[params[2]]
    assert [g["lr"] for g in second.param_groups] == [0.1, 0.2]


@pytest.mark.parametrize("t", TYPES)
def test_what_hooks_see_and_change(t):
    # a hook before the loading may give another state; one after it sees the loaded state
    p = _param((4, 4), t, 0)
    first, second = OrthogonalMomentum([p], lr=0.1), OrthogonalMomentum([p], lr=0.1)
    first.state[p]["momentum_buffer"] = torch.randn(4, 4)

    def doubled(_, state):
        state = copy.deepcopy(state)
        state["state"][0]["momentum_buffer"] *= 2
        return state

    seen = []
    second.register_load_state_dict_pre_hook(doubled)
    second.register_load_state_dict_post_hook(lambda o: seen.append(o.state[p]["momentum_buffer"].dtype))
    second.load_state_dict(first.state_dict())
    assert torch.equal(second.state[p]["momentum_buffer"], 2 * first.state[p]["momentum_buffer"])
    assert seen == [torch.float32]


def test_a_state_that_does_not_fit_is_refused():
    p = _param((4, 4), torch.bfloat16, 0)
    first, second = OrthogonalMomentum([p], lr=0.1), OrthogonalMomentum([p, _param((2, 2), p.dtype, 1)], lr=0.1)
    with pytest.raises(ValueError):
        second.load_state_dict(first.state_dict())


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
def test_a_resumed_training_takes_the_same_steps(gpu, t):
    shapes = [(40, 24), (24, 40), (7, 9)]

    def step(opt, params, k):
        for i, p in enumerate(params):
            p.grad = _param(p.shape, t, 100 * k + i, "cuda").detach()
        opt.step()

    whole = [_param(s, t, i, "cuda") for i, s in enumerate(shapes)]
    opt = OrthogonalMomentum(whole, lr=0.1)
    for k in range(4):
        step(opt, whole, k)
    parts = [_param(s, t, i, "cuda") for i, s in enumerate(shapes)]
    opt = OrthogonalMomentum(parts, lr=0.1)
    for k in range(2):
        step(opt, parts, k)
    resumed = OrthogonalMomentum(parts, lr=0.1)
    resumed.load_state_dict(opt.state_dict())
    for k in range(2, 4):
        step(resumed, parts, k)
    assert all(torch.equal(a, b) for a, b in zip(whole, parts))


@pytest.mark.gpu
@pytest.mark.parametrize("wrong", [lambda b: b.bfloat16(), lambda b: b[:, :3].clone(), lambda b: b.cpu(),
                                   lambda b: b.t().contiguous().t(), lambda b: b.double(), lambda b: None])
def test_a_buffer_that_is_not_the_kernels_is_refused(gpu, wrong):
    p = _param((4, 4), torch.bfloat16, 0, "cuda")
    p.grad = torch.ones_like(p)
    opt = OrthogonalMomentum([p], lr=0.1)
    before = p.detach().clone()
    opt.state[p]["momentum_buffer"] = wrong(torch.zeros((4, 4), device="cuda"))
    with pytest.raises(RuntimeError, match="momentum_buffer"):
        opt.step()
    assert torch.equal(p, before)
