"""Argument checks of the token operators' C entry points: all of them come
before any HIP call, so they run without a device."""
import ctypes as C

import pytest

from blitzgs_amd import _lib, build

NZ = C.c_void_p(256)
F32, BF16, F16 = 0, 1, 2


@pytest.fixture(scope="module")
def lib():
    if build.needs_build():
        build.build(force=True)
    return _lib.load()


def _refused(lib, rc, words):
    assert rc != 0 and words in lib.gs_last_error(), lib.gs_last_error()


def test_layer_norm(lib):
    fwd = lambda type=F32, params=F32, rows=4, width=8, x=NZ, xs=8, eps=1e-5, y=NZ, mean=None: (  # noqa: E731
        lib.gs_layer_norm_forward(type, params, rows, width, x, xs, None, None, eps, y, mean, None, None))
    _refused(lib, fwd(type=3), b"element type")
    _refused(lib, fwd(type=BF16, params=F16), b"parameters")
    _refused(lib, fwd(rows=-1), b"rows")
    _refused(lib, fwd(width=0), b"width")
    _refused(lib, fwd(width=32769, xs=32769), b"width")
    _refused(lib, fwd(xs=7), b"overlap")
    _refused(lib, fwd(x=None), b"non-null")
    _refused(lib, fwd(eps=-1.0), b"eps")
    _refused(lib, fwd(mean=NZ), b"together")
    assert fwd(rows=0) == 0
    bwd = lambda x=NZ, ws=NZ: lib.gs_layer_norm_backward(  # noqa: E731
        F32, F32, 4, 8, x, 8, None, NZ, NZ, NZ, 8, NZ, NZ, NZ, ws, None)
    _refused(lib, bwd(ws=None), b"workspace")
    _refused(lib, bwd(x=None), b"non-null")
    assert lib.gs_layer_norm_workspace_bytes(F32, 4, 0) == 0
    # one partial row of both gradients at least, and no more for many rows than for a full grid
    assert lib.gs_layer_norm_workspace_bytes(F32, 1, 1000) >= 8000
    assert lib.gs_layer_norm_workspace_bytes(F32, 10 ** 9, 1000) <= 2 ** 24


def _strides(*s):
    return (C.c_int64 * 3)(*s)


def test_attention(lib):
    s = _strides(64, 64, 16)

    def fwd(type=BF16, B=1, Hq=2, Hkv=1, Tq=4, Tk=4, D=16, q=NZ, k=NZ, scale=0.25, strides=s):
        return lib.gs_attention_forward(type, B, Hq, Hkv, Tq, Tk, D, q, strides, k, s, NZ, s, scale, 0, None, None, NZ,
                                        s, None, None, None, None)
    _refused(lib, fwd(type=-1), b"element type")
    _refused(lib, fwd(B=-1), b"negative")
    _refused(lib, fwd(Hq=3, Hkv=2), b"multiple")
    _refused(lib, fwd(Hkv=0), b"multiple")
    _refused(lib, fwd(D=0), b"head dimension")
    _refused(lib, fwd(D=129), b"head dimension")
    _refused(lib, fwd(scale=0.0), b"scale")
    _refused(lib, fwd(scale=float("nan")), b"scale")
    _refused(lib, fwd(scale=float("inf")), b"scale")
    _refused(lib, fwd(q=None), b"must be given")
    _refused(lib, fwd(strides=None), b"must be given")
    _refused(lib, fwd(k=None), b"non-null")
    _refused(lib, fwd(Tk=100000), b"workspace")
    _refused(lib, fwd(Hq=2 ** 16, Hkv=1, Tq=2 ** 15), b"too many")
    assert fwd(B=0) == 0 and fwd(Tq=0) == 0

    def bwd(o=NZ, ws=NZ, dk=NZ, Tk=4):
        return lib.gs_attention_backward(BF16, 1, 2, 1, 4, Tk, 16, NZ, s, NZ, s, NZ, s, 0.25, 0, None, None, o, s, None,
                                         NZ, NZ, s, NZ, s, dk, s, NZ, s, ws, None)
    _refused(lib, bwd(ws=None), b"workspace")
    _refused(lib, bwd(o=None), b"non-null")
    _refused(lib, bwd(dk=None), b"together")
    assert lib.gs_attention_workspace_bytes(BF16, 1, 2, 1, 4, 4, 0, 0, 0) == 0
    # one query over many keys is split and needs room for partial results
    assert lib.gs_attention_workspace_bytes(BF16, 1, 1, 1, 1, 100000, 64, 0, 0) >= 2 * 66 * 4


def test_orthogonalise(lib):
    call = lambda type=F32, count=1, m=4, n=4, x=NZ, steps=5, ws=NZ: lib.gs_orthogonalise(  # noqa: E731
        type, count, m, n, x, steps, NZ, ws, None)
    _refused(lib, call(type=5), b"element type")
    _refused(lib, call(count=-1), b"negative")
    _refused(lib, call(count=65536), b"65535")
    _refused(lib, call(m=65537), b"65536")
    _refused(lib, call(steps=0), b"steps")
    _refused(lib, call(steps=33), b"steps")
    _refused(lib, call(x=None), b"non-null")
    _refused(lib, call(ws=C.c_void_p(264)), b"aligned")
    assert call(count=0) == 0 and call(m=0) == 0
    assert lib.gs_orthogonalise_workspace_bytes(1, -1, 4) == 0
    assert lib.gs_orthogonalise_workspace_bytes(2, 100, 200) >= 2 * 8 * (100 * 200 + 100 * 100)
    p = (C.c_void_p * 1)(256)
    none = (C.c_void_p * 1)(None)
    _refused(lib, lib.gs_momentum_update(F32, 33, 4, p, p, 0.9, 1, NZ, None), b"at most 32")
    _refused(lib, lib.gs_momentum_update(F32, 1, 4, none, p, 0.9, 1, NZ, None), b"null tensor")
    _refused(lib, lib.gs_momentum_update(F32, 1, -1, p, p, 0.9, 1, NZ, None), b"size")
    _refused(lib, lib.gs_momentum_apply(F32, 1, 4, none, 1.0, 0.1, NZ, None), b"null tensor")
    _refused(lib, lib.gs_momentum_apply(7, 1, 4, p, 1.0, 0.1, NZ, None), b"element type")
