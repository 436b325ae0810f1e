"""The C entry points refuse pointers between elements: a kernel's access there would fault."""
from __future__ import annotations

import ctypes

import pytest

from guass_b200 import _block, _lib

FAKE = 1 << 20  # an aligned address that no accepted call reaches
BAD = _lib.GF_ERR_INVALID_ARG


def refused(status):
    return status == BAD and "elements" in _lib.last_error()


@pytest.mark.parametrize("name", ["x", "w_in", "b_in", "w_out", "b_out", "y", "dy", "dx", "dw_in", "db_in", "dw_out",
                                  "db_out"])
def test_feed_forward(name):
    f = _block.GfGatedFf(tokens=4, in_features=8, hidden=16, out_features=8, dtype=_lib.GF_BF16, ld_x=8, ld_w_in=8,
                         ld_w_out=16, ld_y=8, ld_dy=8, h=FAKE)
    for n in ("x", "w_in", "w_out", "y", "dy"):
        setattr(f, n, FAKE)
    setattr(f, name, FAKE + 1)
    L = _block.lib()
    for fn in (L.gf_gated_ff_forward, L.gf_gated_ff_backward):
        assert refused(fn(ctypes.byref(f), FAKE, 1 << 20, None))
    assert L.gf_gated_ff_workspace_bytes(ctypes.byref(f), 0) == 0


@pytest.mark.parametrize("dtype,off", [(_lib.GF_F32, 1), (_lib.GF_F32, 2), (_lib.GF_BF16, 1), (_block.GF_F16, 3)])
def test_dropout_and_quantisation(dtype, off):
    L, rule = _block.lib(), _block.GfDropoutRule(p=0.5)
    for x, r, y in ((off, 0, 0), (0, off, 0), (0, 0, off)):
        assert refused(L.gf_dropout(2, 2, dtype, ctypes.byref(rule), FAKE + x, 2, 1, FAKE + r, 2, 1, FAKE + y, None))
    assert refused(L.gf_quantize_rows(2, 4, dtype, FAKE + off, 4, FAKE, 16, FAKE, None))
    assert refused(L.gf_quantize_rows(2, 4, dtype, FAKE, 4, FAKE, 16, FAKE + 2, None))


@pytest.mark.parametrize("name,off", [("a_scale", 2), ("b_scale", 1), ("bias", 1), ("out", 1)])
def test_8_bit_product(name, off):
    L = _block.lib()
    d = dict(m=2, n=2, k=16, dtype=_lib.GF_BF16, a=FAKE, b=FAKE, a_scale=FAKE, b_scale=FAKE, bias=FAKE, out=FAKE, ld_a=16,
             ld_b=16, ld_out=2)
    d[name] += off
    p = _block.GfInt8Product(**d)
    assert refused(L.gf_int8_matmul(ctypes.byref(p), FAKE, 1 << 20, None))
    if name != "a_scale":
        assert refused(L.gf_int8_linear(ctypes.byref(p), FAKE, 16, _lib.GF_BF16, FAKE, 1 << 20, None))
    good = _block.GfInt8Product(**{**d, name: FAKE})
    assert refused(L.gf_int8_linear(ctypes.byref(good), FAKE + 2, 16, _lib.GF_F32, FAKE, 1 << 20, None))


def test_status_copy():
    L = _block.lib()
    assert refused(L.gf_block_status_async(FAKE + 2, None)) and L.gf_block_status_async(None, None) == BAD
