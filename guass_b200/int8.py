"""Linear layers in 8-bit integers: a scale for each token and each output
channel, exact integer sums on the tensor cores.

The serving form of a merged weight ``W0 + delta``: quantise it once
(:func:`quantize_rows`, :class:`Int8Linear`,
:meth:`guass_b200.adapters.BatchedAdapters.quantize_merged`), then
:func:`int8_linear` quantises each call's activations row by row and
multiplies.  Forward only.
"""
from __future__ import annotations

import torch
from torch import nn

from guass_b200 import _block

_MAX_K = 131071


def quantize_rows(x):
    """``(q, scale)``: each row of ``x`` [..., K] (fp32, bf16 or fp16) in 8
    bits, ``scale = max|x| / 127`` and ``q = round(x * (127 / max|x|))`` (to
    even), both in fp32.  A row whose maximum is below 2^-100 gives zeros and
    scale 0; a row that holds an infinity or a NaN gives zeros and scale NaN,
    so that products with it are NaN.  Not differentiable.  ``q`` [..., K] is a view of rows that
    start on 16-byte boundaries, the layout the product reads in place."""
    _block.check_tensor("x", x, tuple(_block.DTYPES))
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError("x needs a last dimension of at least 1")
    k = x.shape[-1]
    v = _block.rows_of(x.detach(), k)
    kp = -(-k // 16) * 16
    q = torch.empty(v.shape[0], kp, dtype=torch.int8, device=x.device)
    scale = torch.empty(v.shape[0], dtype=torch.float32, device=x.device)
    _block.call(x.device, _block.lib().gf_quantize_rows, v.shape[0], k, _block.DTYPES[x.dtype], v.data_ptr(),
                _block.ld(v), q.data_ptr(), kp, scale.data_ptr())
    return q.view(*x.shape[:-1], kp)[..., :k], scale.view(x.shape[:-1])


def _forward_only(who, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{who} has no backward: call it under torch.no_grad() or on detached inputs")
    _block.refuse_tangents(who, *tensors)


def _check_weight(b, b_scale, bias, out_dtype, device):
    """[N, K] int8 with [N] scales and bias: (n, k)."""
    _block.check_tensor("the int8 weight", b, (torch.int8,), device)
    _block.check_tensor("its scales", b_scale, (torch.float32,), device)
    if out_dtype not in _block.DTYPES:
        raise ValueError(f"out_dtype must be one of {list(_block.DTYPES)}, got {out_dtype}")
    if b.dim() != 2:
        raise ValueError(f"the int8 weight must be [N, K], got {tuple(b.shape)}")
    n, k = b.shape
    if n == 0 or not 0 < k <= _MAX_K:
        raise ValueError(f"N must be positive and K in 1..{_MAX_K}, got N={n}, K={k}")
    if b_scale.dim() != 1 or b_scale.shape[0] != n:
        raise ValueError(f"the weight's scales must be [{n}], got {tuple(b_scale.shape)}")
    if bias is not None:
        _block.check_tensor("bias", bias, (out_dtype,), device)
        if bias.dim() != 1 or bias.shape[0] != n:
            raise ValueError(f"bias must be [{n}], got {tuple(bias.shape)}")
    return n, k


def _describe(m, n, k, b, b_scale, bias, out):
    d = _block.GfInt8Product()
    d.m, d.n, d.k, d.dtype = m, n, k, _block.DTYPES[out.dtype]
    d.b, d.ld_b, d.b_scale = b.data_ptr(), _block.ld(b), b_scale.data_ptr()
    if bias is not None:
        d.bias = bias.data_ptr()
    d.out, d.ld_out = out.data_ptr(), n
    return d


def int8_matmul(a, a_scale, b, b_scale, bias=None, *, out_dtype=torch.bfloat16):
    """``(a b^T) * a_scale[:, None] * b_scale + bias`` as ``out_dtype``.

    ``a`` [M, K] and ``b`` [N, K] int8 (K at most 131071, so that the integer
    sums are exact), ``a_scale`` [M] and ``b_scale`` [N] fp32, ``bias`` [N] of
    ``out_dtype`` or None.  Any row strides; rows that do not start on 16-byte
    boundaries cost a copy.  Forward only."""
    _block.check_tensor("a", a, (torch.int8,))
    _block.check_tensor("a_scale", a_scale, (torch.float32,), a.device)
    _forward_only("int8_matmul", a_scale, b_scale, bias)
    n, k = _check_weight(b, b_scale, bias, out_dtype, a.device)
    if a.dim() != 2 or a.shape[1] != k:
        raise ValueError(f"a is {tuple(a.shape)}, b {tuple(b.shape)}: expected [M, K] and [N, K]")
    m = a.shape[0]
    if tuple(a_scale.shape) != (m,):
        raise ValueError(f"a_scale must be [{m}], got {tuple(a_scale.shape)}")
    a, b, a_scale, b_scale = _block.rows_of(a, k), _block.rows_of(b, k), a_scale.contiguous(), b_scale.contiguous()
    bias = None if bias is None else bias.contiguous()
    out = torch.empty(m, n, dtype=out_dtype, device=a.device)
    if m == 0:
        return out
    d = _describe(m, n, k, b, b_scale, bias, out)
    d.a, d.ld_a, d.a_scale = a.data_ptr(), _block.ld(a), a_scale.data_ptr()
    L = _block.lib()
    _block.run(a.device, L.gf_int8_product_workspace_bytes, L.gf_int8_matmul, d)
    return out


def int8_linear(x, q_weight, weight_scale, bias=None, *, out_dtype=None):
    """``linear(x, q_weight * weight_scale[:, None], bias)`` with ``x`` [..., K]
    (fp32, bf16 or fp16) quantised row by row as :func:`quantize_rows` does;
    ``q_weight`` [N, K] int8, ``weight_scale`` [N] fp32, ``bias`` [N] of
    ``out_dtype``, which defaults to ``x``'s.  Forward only: refuses inputs
    that need a gradient."""
    _block.check_tensor("x", x, tuple(_block.DTYPES))
    _forward_only("int8_linear", x, weight_scale, bias)
    out_dtype = x.dtype if out_dtype is None else out_dtype
    n, k = _check_weight(q_weight, weight_scale, bias, out_dtype, x.device)
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"x is {tuple(x.shape)}, q_weight {tuple(q_weight.shape)}: expected [..., K] and [N, K]")
    out = torch.empty(*x.shape[:-1], n, dtype=out_dtype, device=x.device)
    if out.numel() == 0:
        return out
    x, q_weight, weight_scale = _block.rows_of(x, k), _block.rows_of(q_weight, k), weight_scale.contiguous()
    bias = None if bias is None else bias.contiguous()
    d = _describe(x.shape[0], n, k, q_weight, weight_scale, bias, out)
    L = _block.lib()
    _block.run(x.device, L.gf_int8_linear_workspace_bytes, L.gf_int8_linear, d, x.data_ptr(), _block.ld(x),
               _block.DTYPES[x.dtype])
    return out


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

    def _apply(self, fn, recurse=True):
        """Casts (``.half()``, ``.to(torch.bfloat16)``) reach the bias alone: scales stay fp32."""
        scale = self.weight_scale
        super()._apply(fn, recurse)
        if self.weight_scale.dtype != scale.dtype:
            self.weight_scale = scale.to(self.weight_scale.device)
        return self

    def forward(self, x):
        bias = self.bias if self.bias is None or self.bias.dtype == x.dtype else self.bias.to(x.dtype)
        return int8_linear(x, self.q_weight, self.weight_scale, bias)
