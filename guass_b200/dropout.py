"""Dropout from a counter-based generator: the mask is a function of (seed,
site, row, column), so the backward makes it again and nothing is stored."""
from __future__ import annotations

import ctypes

import torch

from guass_b200 import _block


def _rows(t):
    """(tensor, rows, columns, row stride, column stride) of ``t`` as [rows,
    last dimension], whatever its strides (a copy only where its leading
    dimensions cannot be one)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1]) if t.dim() else t.reshape(1, 1)
    return t, *t.shape, *t.stride()


def _run(x, rule, residual):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    x, rows, cols, row_stride, col_stride = _rows(x)
    ptr, r_row, r_col = None, 0, 0
    if residual is not None:
        residual, _, _, r_row, r_col = _rows(residual)
        ptr = residual.data_ptr()
    _block.call(x.device, _block.lib().gf_dropout, rows, cols, _block.DTYPES[x.dtype], ctypes.byref(rule), x.data_ptr(),
                row_stride, col_stride, ptr, r_row, r_col, y.data_ptr())
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, site):
        rule = _block.make_rule(p, seed, site, x.device)
        ctx.kept = _block.KeptRule(rule, seed)
        return _run(x, rule, residual)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        rule = ctx.kept.get(dy.device)
        dx = _run(dy, rule, None) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x, p: float, seed, *, site: int = 0, residual=None):
    """``residual + dropout(x)`` (without ``residual``: ``dropout(x)``).

    Element (r, c) of ``x`` seen as [rows, last dimension] is dropped with
    probability ``p`` (0 <= p < 1) and otherwise multiplied by ``1 / (1 - p)``;
    a dropped element contributes 0 whatever it holds.  ``seed`` is an int, or
    a one-element int64 CUDA tensor that the kernel reads when it runs: a
    captured training step advances it between replays (it must not change
    between a forward and its backward).  ``site`` tells apart the dropouts
    that share a seed: the same (seed, site, shape) always gives the same mask,
    on any device, stream and layout.

    fp32, bf16 or fp16 with any strides; the result is contiguous.
    Differentiable once in ``x`` and ``residual``, in reverse mode."""
    _block.check_tensor("x", x, tuple(_block.DTYPES))
    if residual is not None:
        _block.check_tensor("residual", residual, (x.dtype,), x.device)
        if residual.shape != x.shape:
            raise ValueError(f"residual is {tuple(residual.shape)}, x {tuple(x.shape)}")
    if x.numel() == 0:
        _block.make_rule(p, seed, site, x.device)
        return x.clone() if residual is None else residual + x
    _block.refuse_tangents("dropout", x, residual)
    if torch.is_grad_enabled() and (x.requires_grad or residual is not None and residual.requires_grad):
        return _Dropout.apply(x, residual, p, seed, site)
    return _run(x, _block.make_rule(p, seed, site, x.device), residual)
