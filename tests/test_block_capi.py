"""Argument checks of the C entry points of the rotary, feed-forward and AdamW operators:
all of them come before any HIP call, so they run without a device.  The 8-bit moments'
hash, and what an optimiser's state keeps, on the CPU."""
import copy
import ctypes as C

import pytest
import torch

from blitzgs_amd import _lib, build
from block_helpers import draws

NZ = C.c_void_p(256)
F32, BF16, F16 = 0, 1, 2


@pytest.fixture(scope="module")
def lib():
    if build.needs_build():
        build.build(force=True)
    return _lib.load()


def _refused(lib, rc, words):
    assert rc != 0 and words in lib.gs_last_error(), lib.gs_last_error()


def test_rotary(lib):
    s = (C.c_int64 * 3)(64, 64, 16)

    def fwd(type=BF16, params=BF16, B=1, Hq=2, Hk=1, T=4, D=16, axes=1, pairs=8, norm=1, eps=1e-6, q=NZ, k=NZ, at=NZ):
        return lib.gs_rotary_forward(type, params, B, Hq, Hk, T, D, axes, pairs, 0, 1.0, norm, eps, q, s, k, s, None, None,
                                     at, 0, s, NZ, NZ, s, NZ, s, None)
    _refused(lib, fwd(type=3), b"element type")
    _refused(lib, fwd(params=F16), b"weights")
    _refused(lib, fwd(B=-1), b"negative")
    _refused(lib, fwd(Hq=65537), b"65536 heads")
    for D in (0, 257):
        _refused(lib, fwd(D=D), b"head dimension")
    _refused(lib, fwd(pairs=9), b"do not fit")
    _refused(lib, fwd(pairs=0), b"do not fit")
    _refused(lib, fwd(axes=3, pairs=4), b"do not fit")
    _refused(lib, fwd(axes=2 ** 30, pairs=4), b"do not fit")
    _refused(lib, fwd(eps=-1.0), b"eps")
    _refused(lib, fwd(eps=float("nan")), b"eps")
    _refused(lib, fwd(q=None), b"q, its output")
    _refused(lib, fwd(k=None), b"k, its output")
    _refused(lib, fwd(at=None), b"positions")
    assert fwd(B=0) == 0 and fwd(T=0) == 0 and fwd(Hq=0, Hk=0) == 0

    def bwd(q=NZ, dqy=NZ, dq=NZ, dqw=NZ, ws=NZ, norm=1):
        return lib.gs_rotary_backward(BF16, BF16, 1, 2, 1, 4, 16, 1, 8, 0, 1.0, norm, 1e-6, q, s, NZ, s, None, None, NZ, 0,
                                      s, NZ, dqy, s, NZ, s, dq, s, NZ, s, dqw, None, ws, None)
    _refused(lib, bwd(ws=None), b"workspace")
    _refused(lib, bwd(dqy=None), b"gradients")
    _refused(lib, bwd(q=None), b"gradients")
    _refused(lib, bwd(dq=None), b"comes with its rows")
    assert lib.gs_rotary_workspace_bytes(BF16, 1, 2, 1, 4, 16, 1, 9) == 0
    # a partial row for each workgroup of each side, and no more for many tokens than for a full grid
    assert lib.gs_rotary_workspace_bytes(BF16, 1, 2, 1, 4, 16, 1, 8) >= 2 * 16 * 4
    assert lib.gs_rotary_workspace_bytes(BF16, 1000, 2, 1, 10 ** 6, 16, 1, 8) <= 2 ** 20


def test_feed_forward(lib):
    def fwd(type=BF16, act=0, rows=4, W=8, H=16, O=8, x=NZ, a=None, b=None, rest=None, h=NZ):
        return lib.gs_feed_forward(type, act, rows, W, H, O, x, W, NZ, NZ, NZ, a, b, rest, h, NZ, NZ, None)
    _refused(lib, fwd(type=3), b"element type")
    _refused(lib, fwd(act=2), b"activation")
    _refused(lib, fwd(rows=-1), b"rows")
    _refused(lib, fwd(rows=2 ** 31), b"rows")
    for bad in (dict(W=0), dict(H=0), dict(O=0), dict(H=2 ** 24 + 1)):
        _refused(lib, fwd(**bad), b"width, hidden and out")
    _refused(lib, fwd(a=NZ), b"together")
    _refused(lib, fwd(rest=NZ), b"together")
    _refused(lib, fwd(x=None), b"non-null")
    _refused(lib, fwd(h=None), b"non-null")
    # tiles whose threads are more than a launch takes
    _refused(lib, fwd(rows=2 ** 31 - 2 ** 17, type=F32), b"too many tiles")
    _refused(lib, lib.gs_feed_forward(BF16, 0, 4, 8, 16, 8, NZ, -8, NZ, NZ, NZ, None, None, None, NZ, NZ, NZ, None), b"stride")
    assert fwd(rows=0) == 0

    def bwd(x=NZ, dx=NZ, dd=NZ, ws=NZ, rows=4):
        return lib.gs_feed_forward_backward(BF16, 0, rows, 8, 16, 8, x, 8, NZ, NZ, NZ, NZ, NZ, NZ, NZ, NZ, 8, dx, None, None,
                                            dd, ws, None)
    _refused(lib, bwd(x=None), b"non-null")
    _refused(lib, bwd(ws=None), b"workspace")
    _refused(lib, bwd(ws=C.c_void_p(264)), b"aligned")
    assert bwd(dx=None, dd=None) == 0
    assert lib.gs_feed_forward_workspace_bytes(BF16, 4, 8, 0, 8, 1) == 0
    # the projections' gradients
    assert lib.gs_feed_forward_workspace_bytes(BF16, 100, 8, 16, 8, 1) >= 2 * 100 * 16 * 2


def _settings(lr=0.1, beta1=0.9, beta2=0.999, eps=1e-8, decay=0.0, step=1, seed=0):
    return C.byref(_lib.AdamWSettings(lr, beta1, beta2, eps, decay, step, seed))


def test_adamw(lib):
    p, none = (C.c_void_p * 1)(256), (C.c_void_p * 1)(None)

    def call(type=F32, bits=32, count=1, size=4, params=p, scales=None, how=_settings()):
        return lib.gs_adamw_update(type, bits, count, (C.c_int64 * 1)(size), params, p, p, p, scales, scales, how, None)
    _refused(lib, call(type=7), b"element type")
    _refused(lib, call(bits=16), b"8 or 32")
    _refused(lib, call(count=-1), b"count")
    _refused(lib, call(size=-1), b"size")
    _refused(lib, call(params=none), b"null pointer")
    _refused(lib, call(params=None), b"non-null")
    _refused(lib, call(how=None), b"settings")
    _refused(lib, call(bits=8), b"scales")
    _refused(lib, call(bits=8, scales=none), b"scales")
    for bad, words in ((dict(step=0), b"step"), (dict(beta1=1.0), b"betas"), (dict(beta2=-0.1), b"betas"),
                       (dict(beta1=float("nan")), b"betas"), (dict(lr=-1.0), b"lr"), (dict(eps=float("nan")), b"lr"),
                       (dict(decay=-1.0), b"lr")):
        _refused(lib, call(how=_settings(**bad)), words)
    assert call(count=0) == 0 and call(size=0, params=none) == 0
    # tensors of 4 floats (or codes, with a scale each) that lie on each other, or a gradient on one of them
    def two(bits=32, **moved):
        at = dict(p=(0, 16), g=(0x100, 0x100), m=(0x200, 0x210), v=(0x300, 0x310), ms=(0x400, 0x401), vs=(0x500, 0x501))
        at = {k: (C.c_void_p * 2)(*(0x10000 + a for a in moved.get(k, places))) for k, places in at.items()}
        scales = (at["ms"], at["vs"]) if bits == 8 else (None, None)
        return lib.gs_adamw_update(F32, bits, 2, (C.c_int64 * 2)(4, 4), at["p"], at["g"], at["m"], at["v"], *scales,
                                   _settings(), None)
    for bits, moved in ((32, dict(p=(0, 0))), (32, dict(p=(0, 12))), (32, dict(m=(0x200, 0x1f8))), (32, dict(v=(0x20c, 0x310))),
                        (8, dict(m=(0x200, 0x203))), (8, dict(ms=(0x400, 0x400))), (8, dict(vs=(0x202, 0x500)))):
        _refused(lib, two(bits, **moved), b"twice in a call or overlap")
    for bits, moved in ((32, dict(g=(0, 0x100))), (32, dict(g=(0x100, 0x1f4))), (32, dict(g=(0x21c, 0x100))),
                        (8, dict(g=(0x100, 0x3f4))), (8, dict(g=(0x1f0, 0x1f1)))):
        rc = two(bits, **moved)
        _refused(lib, rc, b"overlaps")
    values = lambda type=F32, n=4, m=NZ: lib.gs_adamw_values(type, n, m, NZ, NZ, NZ, NZ, NZ, None)  # noqa: E731
    _refused(lib, values(type=F16), b"float32 or bfloat16")
    _refused(lib, values(n=-1), b"size")
    _refused(lib, values(m=None), b"non-null")
    assert values(n=0) == 0


def test_the_rounding_bits_are_even():
    # n draws of 16 bits, both halves, their neighbours and steps: means of uniform numbers are within five
    # deviations (0.289 / sqrt(n)) of 1/2 and correlations of 0 (1 / sqrt(n))
    n = 1 << 18
    one = draws(n, 0, 1, 0)
    parts = [one & 65535, one >> 16, draws(n, 1, 1, 0) & 65535, draws(n, 0, 2, 0) & 65535, draws(n, 0, 1, 1) & 65535]
    u = torch.stack([p.double() / 65536 for p in parts])
    assert (u.mean(1) - 0.5).abs().max() < 5 * 0.289 / n ** 0.5
    c = (u - 0.5) / 0.2887
    # the squares' own deviation is 0.9 / sqrt(n)
    assert ((c @ c.T / n) - torch.eye(len(parts))).abs().max() < 5 / n ** 0.5
    for lag in (1, 2, 8, 128, 2048):
        assert (c[:, lag:] * c[:, :-lag]).mean(1).abs().max() < 5 / (n - lag) ** 0.5
    assert len(torch.unique(one)) > 0.999 * n


def test_a_state_keeps_its_types():
    from blitzgs_amd.adamw import AdamW
    p = torch.nn.Parameter(torch.randn(10, 30).bfloat16())
    for bits in (8, 32):
        first, second = AdamW([p], bits=bits), AdamW([p], bits=bits)
        moment = (lambda *s: torch.randint(0, 100, s).to(torch.uint8)) if bits == 8 else torch.randn
        first.state[p].update(step=7, exp_avg=moment(10, 30), exp_avg_sq=moment(10, 30))
        if bits == 8:
            first.state[p]["scales"] = moment(2, 3)
        second.load_state_dict(copy.deepcopy(first.state_dict()))
        assert second.state[p]["step"] == 7 and set(second.state[p]) == set(first.state[p])
        for name, want in first.state[p].items():
            if name != "step":
                got = second.state[p][name]
                assert got.dtype == want.dtype and torch.equal(got, want) and got.data_ptr() != want.data_ptr()
