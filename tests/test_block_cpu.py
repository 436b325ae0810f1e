"""Host side of the block operators (no GPU): the C ABI, argument checks, the
reference generator."""
from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

import block_reference as ref
from guass_b200 import _block, _lib
from guass_b200.dropout import dropout
from guass_b200.feedforward import gated_feed_forward
from guass_b200.int8 import int8_linear, int8_matmul, quantize_rows

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "gfblock.h"
FAKE = 1 << 20  # an aligned address that no accepted call reaches


def test_header_library_and_binding_agree():
    declared = set(re.findall(r"^\s*[\w\s\*]*?\b(gf_\w+)\s*\(", HEADER.read_text(), flags=re.M))
    assert declared == set(_block.EXPORTED)
    for name in declared:
        assert hasattr(_block.lib(), name), name


def test_struct_layout_matches_c(tmp_path):
    structs = {"gf_dropout_rule": _block.GfDropoutRule, "gf_gated_ff": _block.GfGatedFf,
               "gf_int8_product": _block.GfInt8Product}
    body = "".join(f'printf("{c} %zu\\n", sizeof({c}));' + "".join(
        f'printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for f, _ in t._fields_) for c, t in structs.items())
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gfblock.h"\nint main(void) {' + body + "return 0;}")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout
    for line in out.splitlines():
        name, value = line.rsplit(" ", 1)
        c, _, field = name.partition(".")
        want = getattr(structs[c], field).offset if field else ctypes.sizeof(structs[c])
        assert want == int(value), name


def _ff(**kw):
    f = _block.GfGatedFf(tokens=4, in_features=8, hidden=16, out_features=8, dtype=_lib.GF_BF16, ld_x=8, ld_w_in=8,
                         ld_w_out=16, ld_y=8, ld_dy=8)
    for name in ("x", "w_in", "w_out", "h", "y", "dy"):
        setattr(f, name, FAKE)
    for k, v in kw.items():
        setattr(f.dropout if k in ("p", "reserved", "seed_ptr") else f, k, v)
    return f


@pytest.mark.parametrize("kw,status,msg", [
    (dict(hidden=0), _lib.GF_ERR_INVALID_ARG, "positive"),
    (dict(tokens=-1), _lib.GF_ERR_INVALID_ARG, "positive"),
    (dict(tokens=1 << 31), _lib.GF_ERR_UNSUPPORTED, "2\\^31"),
    (dict(hidden=1 << 30, ld_w_out=1 << 30), _lib.GF_ERR_UNSUPPORTED, "2\\^31"),
    (dict(dtype=_lib.GF_F32), _lib.GF_ERR_UNSUPPORTED, "dtype"),
    (dict(activation=2), _lib.GF_ERR_INVALID_ARG, "activation"),
    (dict(ld_x=7), _lib.GF_ERR_INVALID_ARG, "leading dimension"),
    (dict(p=1.0), _lib.GF_ERR_INVALID_ARG, r"\[0, 1\)"),
    (dict(p=float("nan")), _lib.GF_ERR_INVALID_ARG, r"\[0, 1\)"),
    (dict(reserved=1), _lib.GF_ERR_INVALID_ARG, "reserved"),
    (dict(seed_ptr=FAKE + 4), _lib.GF_ERR_INVALID_ARG, "seed_ptr"),
])
def test_feed_forward_descriptions_refused(kw, status, msg):
    L = _block.lib()
    f = _ff(**kw)
    for fn in (L.gf_gated_ff_forward, L.gf_gated_ff_backward):
        assert fn(ctypes.byref(f), FAKE, 1 << 20, None) == status
        assert re.search(msg, _lib.last_error())
    assert L.gf_gated_ff_workspace_bytes(ctypes.byref(f), 0) == 0


def test_feed_forward_pointers_and_workspace_refused():
    L = _block.lib()

    def forward(ws=FAKE, size=1 << 20, **kw):
        return L.gf_gated_ff_forward(ctypes.byref(_ff(**kw)), ws, size, None), _lib.last_error()

    def backward(ws=FAKE, size=1 << 20, **kw):
        return L.gf_gated_ff_backward(ctypes.byref(_ff(dx=FAKE, **kw)), ws, size, None), _lib.last_error()

    bad = _lib.GF_ERR_INVALID_ARG
    for name in ("x", "w_in", "w_out", "h", "y"):
        assert forward(**{name: None}) == (bad, "gf_gated_ff_forward: x, w_in, w_out, h and y must be non-null")
    assert forward(h=FAKE + 8)[0] == bad and "16-byte" in _lib.last_error()
    assert forward(ws=None)[0] == bad and "256-byte" in _lib.last_error()
    assert forward(ws=FAKE + 16)[0] == bad
    assert forward(size=16)[0] == bad and "too small" in _lib.last_error()
    assert forward(ld_y=7)[0] == bad
    for name in ("dy", "w_out", "x", "w_in"):
        assert backward(**{name: None})[0] == bad
    assert backward(size=16)[0] == bad and "too small" in _lib.last_error()
    assert backward(ld_dy=7)[0] == bad
    assert L.gf_gated_ff_forward(None, FAKE, 1 << 20, None) == bad
    assert forward(tokens=0, x=None) == (_lib.GF_OK, _lib.last_error())  # nothing to do


def test_workspace_covers_unaligned_copies():
    L = _block.lib()
    plain = L.gf_gated_ff_workspace_bytes(ctypes.byref(_ff(hidden=64, ld_w_out=64)), 0)
    odd = L.gf_gated_ff_workspace_bytes(ctypes.byref(_ff(hidden=64, ld_w_out=65, ld_x=9, ld_w_in=9)), 0)
    assert plain == 256  # nothing to copy: the least a call takes
    assert odd >= 2 * 4 * 8 + 2 * 128 * 8 + 2 * 8 * 64  # x, w_in and w_out


def test_dropout_and_int8_descriptions_refused():
    L = _block.lib()
    rule = _block.GfDropoutRule(p=0.5)

    def drop(rows=2, cols=2, dtype=0, rule=rule, x=FAKE, y=FAKE):
        return L.gf_dropout(rows, cols, dtype, None if rule is None else ctypes.byref(rule), x, 2, 1, None, 0, 0, y, None)

    bad, no = _lib.GF_ERR_INVALID_ARG, _lib.GF_ERR_UNSUPPORTED
    assert drop(rows=-1) == bad and drop(x=None) == bad and drop(y=None) == bad and drop(rule=None) == bad
    assert drop(rule=_block.GfDropoutRule(p=-0.1)) == bad
    assert drop(dtype=3) == no and drop(cols=1 << 34) == no and drop(rows=1 << 61, cols=4) == no
    assert drop(rows=0, x=None) == _lib.GF_OK

    def quant(rows=2, cols=4, dtype=0, x=FAKE, ld_x=4, ld_q=16):
        return L.gf_quantize_rows(rows, cols, dtype, x, ld_x, FAKE, ld_q, FAKE, None)

    assert quant(cols=0) == bad and quant(x=None) == bad and quant(ld_x=3) == bad and quant(ld_q=3) == bad
    assert quant(dtype=7) == no and quant(cols=1 << 31, ld_x=1 << 31, ld_q=1 << 31) == no
    assert quant(rows=0, x=None) == _lib.GF_OK

    def product(ws=FAKE, size=1 << 20, **kw):
        d = dict(m=2, n=2, k=16, a=FAKE, b=FAKE, a_scale=FAKE, b_scale=FAKE, out=FAKE, ld_a=16, ld_b=16, ld_out=2)
        return L.gf_int8_matmul(ctypes.byref(_block.GfInt8Product(**{**d, **kw})), ws, size, None)

    assert product(n=0) == bad and product(k=0) == bad and product(a=None) == bad and product(ld_a=15) == bad
    assert product(reserved=1) == bad and product(ld_out=1) == bad and product(ws=None) == bad
    assert product(size=8) == bad and "too small" in _lib.last_error()
    assert product(k=131072, ld_a=131072, ld_b=131072) == no and product(dtype=9) == no and product(m=1 << 31) == no
    assert product(m=0, a=None) == _lib.GF_OK

    def linear(ws=FAKE, size=1 << 20, x=FAKE, ld_x=16, x_dtype=0, **kw):
        d = dict(m=2, n=2, k=16, b=FAKE, b_scale=FAKE, out=FAKE, ld_b=16, ld_out=2)
        return L.gf_int8_linear(ctypes.byref(_block.GfInt8Product(**{**d, **kw})), x, ld_x, x_dtype, ws, size, None)

    assert linear(x=None) == bad and linear(ld_x=15) == bad and linear(b=None) == bad and linear(size=256) == bad
    assert linear(x_dtype=5) == no and linear(ws=None) == bad and linear(m=0, x=None) == _lib.GF_OK
    assert L.gf_block_status(None, 0, None) == bad


def test_python_entry_points_refuse_cpu_tensors_and_wrong_types():
    x = torch.zeros(2, 4, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        gated_feed_forward(x, x, x)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        dropout(x, 0.5, 1)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        quantize_rows(x)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        int8_linear(x, x, x)
    with pytest.raises(TypeError, match="torch.Tensor"):
        int8_matmul([1], None, None, None)
    for p in (-0.1, 1.0, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            _block.make_rule(p, 0, 0, None)
    with pytest.raises(ValueError, match="site"):
        _block.make_rule(0.1, 0, 1 << 32, None)
    rule = _block.make_rule(0.1, -1, 3, None)
    assert (rule.seed, rule.site) == (0xFFFFFFFFFFFFFFFF, 3)


def test_row_views():
    t = torch.arange(24.).view(4, 6)
    assert _block.rows_of(t[:, 1:4], 3).data_ptr() == t[:, 1:4].data_ptr()
    for odd in (t.t(), t[:1].expand(4, 6), t.flip(1)):
        v = _block.rows_of(odd, odd.shape[1])
        assert v.is_contiguous() and torch.equal(v, odd)
    assert _block.ld(t[:1, :3]) == 3 and _block.ld(t[:, :3]) == 6


@pytest.mark.parametrize("counter,key,words", [
    # the published known answers of Philox-4x32-10
    ([0] * 4, [0] * 2, [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
    ([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2, [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
    ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0],
     [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]),
])
def test_reference_generator(counter, key, words):
    assert ref.philox(counter, key) == words


def test_reference_mask_is_the_generator():
    keep = ref.keep_mask(3, 10, 0.4, 0x123456789, 6)
    for r in range(3):
        for c in range(10):
            w = ref.philox([c // 4, r, 6, 0], [0x23456789, 0x1])[c % 4]
            assert bool(keep[r, c]) == (w >= round(0.4 * 2 ** 32))


def test_model_options():
    from guass_b200 import sd15

    with pytest.raises(ValueError, match="feed_forward"):
        sd15.UNetConfig(feed_forward="fast")
    with pytest.raises(ValueError, match="dropout"):
        sd15.UNetConfig(dropout=1.0)
    model = sd15.SD15UNet(sd15.tiny_config(), dtype=torch.float32)
    assert model.dropout_seed is None and "dropout_seed" not in model.state_dict()
    cfg = sd15.tiny_config()
    cfg.feed_forward = "kernel"
    blk = sd15.TransformerBlock(32, cfg, lambda i, o, b: torch.nn.Linear(i, o, b))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        blk.feed_forward(torch.zeros(1, 2, 32, dtype=torch.bfloat16))
