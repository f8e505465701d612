"""Attention's scale at the end of its range, where the check comes before any HIP
call: so it runs without a device."""
import ctypes as C

import pytest

from blitzgs_amd import _lib, build

NZ = C.c_void_p(256)


@pytest.fixture(scope="module")
def lib():
    if build.needs_build():
        build.build(force=True)
    return _lib.load()


# the kernels take scale log2(e), which has to be finite too
@pytest.mark.parametrize("scale,fits", [(2.3e38, True), (2.4e38, False), (3e38, False), (3.4e38, False),
                                        (1e-38, True), (0.0, False)])
def test_the_scale_in_powers_of_two_is_finite(lib, scale, fits):
    s = (C.c_int64 * 3)(64, 64, 16)
    # no batch: nothing is launched
    rc = lib.gs_attention_forward(1, 0, 2, 1, 4, 4, 16, NZ, s, NZ, s, NZ, s, scale, 0, None, None, NZ, s, None, None,
                                  None, None)
    assert rc == 0 if fits else rc != 0 and b"scale" in lib.gs_last_error()
    rc = lib.gs_attention_backward(1, 0, 2, 1, 4, 4, 16, NZ, s, NZ, s, NZ, s, scale, 0, None, None, NZ, s, None, NZ, NZ,
                                   s, NZ, s, NZ, s, NZ, s, NZ, None)
    assert rc == 0 if fits else rc != 0 and b"scale" in lib.gs_last_error()
