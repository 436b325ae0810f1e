"""ctypes binding of the block operators in libgfield.so (include/gfblock.h)
and the checks their Python entry points share."""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from guass_b200 import _lib

GF_F16 = 2
GF_FLAG_TIMEOUT = 0x10
ACTIVATIONS = {"gelu": 0, "silu": 1}
DTYPES = {torch.float32: _lib.GF_F32, torch.bfloat16: _lib.GF_BF16, torch.float16: GF_F16}

# Every symbol include/gfblock.h declares.
EXPORTED = ("gf_gated_ff_workspace_bytes", "gf_gated_ff_forward", "gf_gated_ff_backward", "gf_dropout",
            "gf_quantize_rows", "gf_int8_product_workspace_bytes", "gf_int8_matmul",
            "gf_int8_linear_workspace_bytes", "gf_int8_linear", "gf_block_status", "gf_block_status_async")


class GfDropoutRule(ctypes.Structure):
    _fields_ = [
        ("p", ctypes.c_double),
        ("seed", ctypes.c_uint64),
        ("seed_ptr", ctypes.c_void_p),
        ("site", ctypes.c_uint32),
        ("reserved", ctypes.c_uint32),
    ]


class GfGatedFf(ctypes.Structure):
    _fields_ = [
        ("tokens", ctypes.c_int64),
        ("in_features", ctypes.c_int64),
        ("hidden", ctypes.c_int64),
        ("out_features", ctypes.c_int64),
        ("dtype", ctypes.c_int32),
        ("activation", ctypes.c_int32),
        ("dropout", GfDropoutRule),
        ("x", ctypes.c_void_p), ("ld_x", ctypes.c_int64),
        ("w_in", ctypes.c_void_p), ("ld_w_in", ctypes.c_int64),
        ("b_in", ctypes.c_void_p),
        ("w_out", ctypes.c_void_p), ("ld_w_out", ctypes.c_int64),
        ("b_out", ctypes.c_void_p),
        ("h", ctypes.c_void_p),
        ("y", ctypes.c_void_p), ("ld_y", ctypes.c_int64),
        ("dy", ctypes.c_void_p), ("ld_dy", ctypes.c_int64),
        ("dx", ctypes.c_void_p),
        ("dw_in", ctypes.c_void_p),
        ("db_in", ctypes.c_void_p),
        ("dw_out", ctypes.c_void_p),
        ("db_out", ctypes.c_void_p),
    ]


class GfInt8Product(ctypes.Structure):
    _fields_ = [
        ("m", ctypes.c_int64),
        ("n", ctypes.c_int64),
        ("k", ctypes.c_int64),
        ("dtype", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
        ("a", ctypes.c_void_p), ("ld_a", ctypes.c_int64),
        ("b", ctypes.c_void_p), ("ld_b", ctypes.c_int64),
        ("a_scale", ctypes.c_void_p),
        ("b_scale", ctypes.c_void_p),
        ("bias", ctypes.c_void_p),
        ("out", ctypes.c_void_p), ("ld_out", ctypes.c_int64),
    ]


_ready = None


def lib() -> ctypes.CDLL:
    """libgfield.so with the block operators' signatures."""
    global _ready
    if _ready is not None:
        return _ready
    L = _lib.lib()
    i64, i32, ptr, size = ctypes.c_int64, ctypes.c_int32, ctypes.c_void_p, ctypes.c_size_t
    ff = ctypes.POINTER(GfGatedFf)
    L.gf_gated_ff_workspace_bytes.argtypes = [ff, ctypes.c_int]
    L.gf_gated_ff_workspace_bytes.restype = size
    for fn in (L.gf_gated_ff_forward, L.gf_gated_ff_backward):
        fn.argtypes = [ff, ptr, size, ptr]
        fn.restype = ctypes.c_int
    L.gf_dropout.argtypes = [i64, i64, i32, ctypes.POINTER(GfDropoutRule), ptr, i64, i64, ptr, i64, i64, ptr, ptr]
    L.gf_dropout.restype = ctypes.c_int
    L.gf_quantize_rows.argtypes = [i64, i64, i32, ptr, i64, ptr, i64, ptr, ptr]
    L.gf_quantize_rows.restype = ctypes.c_int
    prod = ctypes.POINTER(GfInt8Product)
    L.gf_int8_product_workspace_bytes.argtypes = [prod]
    L.gf_int8_product_workspace_bytes.restype = size
    L.gf_int8_matmul.argtypes = [prod, ptr, size, ptr]
    L.gf_int8_matmul.restype = ctypes.c_int
    L.gf_int8_linear_workspace_bytes.argtypes = [prod]
    L.gf_int8_linear_workspace_bytes.restype = size
    L.gf_int8_linear.argtypes = [prod, ptr, i64, i32, ptr, size, ptr]
    L.gf_int8_linear.restype = ctypes.c_int
    L.gf_block_status.argtypes = [ptr, ctypes.c_int, ctypes.POINTER(ctypes.c_uint32)]
    L.gf_block_status.restype = ctypes.c_int
    L.gf_block_status_async.argtypes = [ptr, ptr]
    L.gf_block_status_async.restype = ctypes.c_int
    _ready = L
    return L


def device_flags(device="cuda", reset: bool = False) -> int:
    """Condition bits the block operators set on ``device`` since the last
    reset (GF_FLAG_TIMEOUT: an output is not valid).  Synchronises the
    current stream."""
    flags = ctypes.c_uint32(0)
    with torch.cuda.device(device):
        _lib.check(lib().gf_block_status(torch.cuda.current_stream().cuda_stream, int(reset), ctypes.byref(flags)))
    return flags.value


class FlagWatch:
    """The condition bits of a device for a loop that does not synchronise:
    :meth:`look` enqueues a copy of them behind the work so far, :meth:`check`
    raises once a copy that has arrived shows one.  (The bits stay set until
    they are reset, so whichever copy arrived last shows them.)"""

    def __init__(self, device: torch.device):
        self.there = torch.zeros(1, dtype=torch.int32, device=device)
        self.flags = torch.zeros(1, dtype=torch.int32, pin_memory=True)

    def look(self) -> None:
        call(self.there.device, lib().gf_block_status_async, self.there.data_ptr())
        # (torch's copy: its allocators keep both ends until it has run, this object gone or not)
        self.flags.copy_(self.there, non_blocking=True)

    def check(self) -> None:
        if self.flags[0] != 0:
            raise RuntimeError(f"a block operator gave up waiting for its own copies or products (condition bits "
                               f"{int(self.flags[0]):#x}): what it computed is not valid")


def check_tensor(name: str, t, dtypes, device=None) -> None:
    """A CUDA tensor of one of ``dtypes`` (and on ``device``)."""
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in dtypes and (device is None or t.device == device):
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t)!r}")
    if t.device.type != "cuda":
        raise RuntimeError(f"{name} must be a CUDA tensor (there is no CPU implementation), got {t.device}")
    if device is not None and t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, the input on {device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")


def refuse_tangents(who: str, *tensors) -> None:
    """Forward-mode derivatives would be lost without a word."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                              for t in tensors):
        raise NotImplementedError(f"{who} has no forward-mode derivative: call it on primals")


def call(device, fn, *args) -> None:
    """``fn(*args, stream)`` on the current stream of ``device`` with that
    device current.  (The raw calls behind torch.cuda.current_stream and
    torch.cuda.device: those objects cost more than a small launch.)"""
    index = device.index
    if index == torch._C._cuda_getDevice():
        _lib.check(fn(*args, torch._C._cuda_getCurrentRawStream(index)))
    else:
        with torch.cuda.device(index):
            _lib.check(fn(*args, torch._C._cuda_getCurrentRawStream(index)))


def run(device, size_fn, fn, desc, *args, room: int = 0, use_room=None, query=()) -> None:
    """``fn(desc, *args, workspace, bytes, stream)`` with the workspace that
    ``size_fn(desc, *query)`` asks for, on ``device`` as :func:`call`.
    ``use_room(pointer)`` gets ``room`` further bytes behind it."""
    index = device.index
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return run(device, size_fn, fn, desc, *args, room=room, use_room=use_room, query=query)
    ref = ctypes.byref(desc)
    n = size_fn(ref, *query)
    if n == 0:
        raise _lib.GfieldError(_lib.GF_ERR_INVALID_ARG, _lib.last_error())
    ws = torch.empty(n + room, dtype=torch.uint8, device=device)
    ptr = ws.data_ptr()
    if use_room is not None:
        use_room(ptr + n)
    _lib.check(fn(ref, *args, ptr, n, torch._C._cuda_getCurrentRawStream(index)))


def rows_of(t: torch.Tensor, cols: int) -> torch.Tensor:
    """``t`` as [rows, cols] with unit column stride and rows that do not
    overlap: a view where its strides allow one, else a copy."""
    v = t if t.dim() == 2 else t.reshape(-1, cols)
    row, col = v.stride()
    if cols > 1 and col != 1 or v.shape[0] > 1 and row < cols:
        v = v.contiguous()
    return v


def ld(v: torch.Tensor) -> int:
    """Leading dimension of a [rows, cols] view."""
    return v.stride(0) if v.shape[0] > 1 else v.shape[1]


class KeptRule:
    """A forward's dropout rule for its backward.  A seed tensor is kept
    itself, not through save_for_backward: under saved-tensor hooks
    (checkpointing, offloading) that would neither keep its memory nor see
    that it changed."""

    __slots__ = ("rule", "seed", "version")

    def __init__(self, rule: GfDropoutRule, seed):
        self.rule, self.seed = rule, seed if isinstance(seed, torch.Tensor) else None
        self.version = None if self.seed is None else seed._version

    def get(self, device) -> GfDropoutRule:
        if self.seed is not None:
            check_tensor("seed", self.seed, (torch.int64,), device)  # its .data may be another tensor's by now
            if self.seed._version != self.version:
                raise RuntimeError("the dropout seed has been modified by an inplace operation between the forward and "
                                   "its backward")
            self.rule.seed_ptr = self.seed.data_ptr()
        return self.rule


def make_rule(p: float, seed, site: int, device) -> GfDropoutRule:
    """``seed``: an int, or a one-element int64 CUDA tensor that the kernel reads."""
    p, site = float(p), int(site)
    if not 0.0 <= p < 1.0:
        raise ValueError(f"dropout probability must be in [0, 1), got {p}")
    if not 0 <= site < 1 << 32:
        raise ValueError(f"site must be in [0, 2**32), got {site}")
    if isinstance(seed, torch.Tensor):
        check_tensor("seed", seed, (torch.int64,), device)
        if seed.numel() != 1:
            raise ValueError(f"a seed tensor has one element, got {tuple(seed.shape)}")
        return GfDropoutRule(p, 0, seed.data_ptr(), site, 0)
    return GfDropoutRule(p, int(seed) & 0xFFFFFFFFFFFFFFFF, None, site, 0)
