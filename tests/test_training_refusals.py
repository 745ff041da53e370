"""What the training operators' entry points refuse on the host, before any launch."""

import ctypes as C

from tileccl_amd import _lib


def refused(rc, text, code=None):
    assert rc == (_lib.ERR_INVALID if code is None else code)
    assert text in _lib.last_error()


def test_two_outputs_in_one_place(lib):
    d = _lib.NormDesc(x=0x1000, residual=0x2000, summed=0x3000, out=0x3000, mean=0x4000, rstd=0x5000, ld_x=64, ld_residual=64, ld_summed=64, ld_out=64,
                      rows=4, cols=64, dtype=_lib.BF16, affine_dtype=_lib.BF16)
    refused(lib.tccl_layer_norm(C.byref(d), None), "out and summed are the same memory")
