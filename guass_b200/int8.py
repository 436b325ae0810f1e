"""Linear layers in 8-bit integers: a scale for each token and each output
channel, exact integer sums on the tensor cores.

The serving form of a merged weight ``W0 + delta``: quantise it once
(:func:`quantize_rows`, :class:`Int8Linear`,
:meth:`guass_b200.adapters.BatchedAdapters.quantize_merged`), then
:func:`int8_linear` quantises each call's activations row by row and
multiplies.  Forward only.
"""
from __future__ import annotations

import ctypes

import torch
from torch import nn

from guass_b200 import _block, _lib

_MAX_K = 131071


def quantize_rows(x):
    """``(q, scale)``: each row of ``x`` [..., K] (fp32, bf16 or fp16) in 8
    bits, ``scale = max|x| / 127`` and ``q = round(x * (127 / max|x|))`` (to
    even), both in fp32.  A row whose maximum is below 2^-100 gives zeros and
    scale 0; a row that holds an infinity or a NaN gives zeros and scale NaN,
    so that products with it are NaN.  ``q`` [..., K] is a view of rows that
    start on 16-byte boundaries, the layout the product reads in place."""
    _block.check_tensor("x", x, tuple(_block.DTYPES))
    _block.require(x.dim() >= 1 and x.shape[-1] > 0, "x needs a last dimension of at least 1")
    k = x.shape[-1]
    v = _block.rows_of(x.detach(), k)
    kp = -(-k // 16) * 16
    q = torch.empty(v.shape[0], kp, dtype=torch.int8, device=x.device)
    scale = torch.empty(v.shape[0], dtype=torch.float32, device=x.device)
    with _block.on_device(x):
        _lib.check(_block.lib().gf_quantize_rows(v.shape[0], k, _block.DTYPES[x.dtype], v.data_ptr(), _block.ld(v),
                                                 q.data_ptr(), kp, scale.data_ptr(),
                                                 torch.cuda.current_stream(x.device).cuda_stream))
    return q.view(*x.shape[:-1], kp)[..., :k], scale.view(x.shape[:-1])


def int8_matmul(a, a_scale, b, b_scale, bias=None, *, out_dtype=torch.bfloat16):
    """``(a b^T) * a_scale[:, None] * b_scale + bias`` as ``out_dtype``.

    ``a`` [M, K] and ``b`` [N, K] int8 (K at most 131071, so that the integer
    sums are exact), ``a_scale`` [M] and ``b_scale`` [N] fp32, ``bias`` [N] of
    ``out_dtype`` or None.  Any row strides; rows that do not start on 16-byte
    boundaries cost a copy."""
    _block.check_tensor("a", a, (torch.int8,))
    _block.check_tensor("b", b, (torch.int8,), a.device)
    _block.check_tensor("a_scale", a_scale, (torch.float32,), a.device)
    _block.check_tensor("b_scale", b_scale, (torch.float32,), a.device)
    _block.require(out_dtype in _block.DTYPES, f"out_dtype must be one of {list(_block.DTYPES)}, got {out_dtype}")
    _block.require(a.dim() == 2 and b.dim() == 2 and a.shape[1] == b.shape[1],
                   f"a is {tuple(a.shape)}, b {tuple(b.shape)}: expected [M, K] and [N, K]")
    m, k = a.shape
    n = b.shape[0]
    _block.require(n > 0 and 0 < k <= _MAX_K, f"N must be positive and K in 1..{_MAX_K}, got N={n}, K={k}")
    _block.require(tuple(a_scale.shape) == (m,) and tuple(b_scale.shape) == (n,), "a_scale must be [M], b_scale [N]")
    if bias is not None:
        _block.check_tensor("bias", bias, (out_dtype,), a.device)
        _block.require(tuple(bias.shape) == (n,), "bias must be [N]")
        bias = bias.contiguous()
    a, b, a_scale, b_scale = _block.rows_of(a, k), _block.rows_of(b, k), a_scale.contiguous(), b_scale.contiguous()
    out = torch.empty(m, n, dtype=out_dtype, device=a.device)
    if m == 0:
        return out
    d = _block.GfInt8Product()
    d.m, d.n, d.k, d.dtype = m, n, k, _block.DTYPES[out_dtype]
    d.a, d.ld_a, d.b, d.ld_b = a.data_ptr(), _block.ld(a), b.data_ptr(), _block.ld(b)
    d.a_scale, d.b_scale = a_scale.data_ptr(), b_scale.data_ptr()
    d.bias = bias.data_ptr() if bias is not None else None
    d.out, d.ld_out = out.data_ptr(), n
    L = _block.lib()
    with _block.on_device(a):
        size = L.gf_int8_product_workspace_bytes(ctypes.byref(d))
        if size == 0:
            raise _lib.GfieldError(_lib.GF_ERR_INVALID_ARG, _lib.last_error())
        ws = torch.empty(size, dtype=torch.uint8, device=a.device)
        _lib.check(L.gf_int8_matmul(ctypes.byref(d), ws.data_ptr(), size,
                                    torch.cuda.current_stream(a.device).cuda_stream))
    return out


def int8_linear(x, q_weight, weight_scale, bias=None, *, out_dtype=None):
    """``linear(x, q_weight * weight_scale[:, None], bias)`` with ``x`` [..., K]
    quantised row by row (:func:`quantize_rows`); ``out_dtype`` defaults to
    ``x``'s.  Forward only: refuses an ``x`` that needs a gradient."""
    _block.check_tensor("x", x, tuple(_block.DTYPES))
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError("int8_linear has no backward: call it under torch.no_grad() or on a detached input")
    _block.check_tensor("q_weight", q_weight, (torch.int8,), x.device)
    _block.require(x.dim() >= 1 and q_weight.dim() == 2 and x.shape[-1] == q_weight.shape[1],
                   f"x is {tuple(x.shape)}, q_weight {tuple(q_weight.shape)}: expected [..., K] and [N, K]")
    q, scale = quantize_rows(x)
    y = int8_matmul(q.reshape(-1, q.shape[-1]), scale.reshape(-1), q_weight, weight_scale, bias,
                    out_dtype=x.dtype if out_dtype is None else out_dtype)
    return y.view(*x.shape[:-1], q_weight.shape[0])


class Int8Linear(nn.Module):
    """A linear layer held in 8 bits: ``Int8Linear.from_weight(weight, bias)``
    quantises a weight [N, K] once, row by row."""

    def __init__(self, q_weight, weight_scale, bias=None):
        super().__init__()
        self.out_features, self.in_features = q_weight.shape
        self.register_buffer("q_weight", q_weight)
        self.register_buffer("weight_scale", weight_scale)
        self.register_buffer("bias", bias)

    @classmethod
    @torch.no_grad()
    def from_weight(cls, weight, bias=None) -> "Int8Linear":
        q, scale = quantize_rows(weight)
        return cls(q, scale, None if bias is None else bias.detach().clone())

    def forward(self, x):
        bias = self.bias if self.bias is None or self.bias.dtype == x.dtype else self.bias.to(x.dtype)
        return int8_linear(x, self.q_weight, self.weight_scale, bias)
