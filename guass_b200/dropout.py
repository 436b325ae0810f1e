"""Dropout from a counter-based generator: the mask is a function of (seed,
site, row, column), so the backward makes it again and nothing is stored."""
from __future__ import annotations

import ctypes

import torch

from guass_b200 import _block, _lib


def _run(x, p, seed, site, residual):
    rule = _block.GfDropoutRule()
    _block.fill_rule(rule, p, seed, site, x.device)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    r = residual if residual is not None else x
    with _block.on_device(x):
        _lib.check(_block.lib().gf_dropout(
            x.shape[0], x.shape[1], _block.DTYPES[x.dtype], ctypes.byref(rule), x.data_ptr(), *x.stride(),
            residual.data_ptr() if residual is not None else None, *r.stride(), y.data_ptr(),
            torch.cuda.current_stream(x.device).cuda_stream))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, site):
        on_device = isinstance(seed, torch.Tensor)
        ctx.save_for_backward(seed if on_device else None)
        ctx.rule = (p, None if on_device else seed, site)
        return _run(x, p, seed, site, residual)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        seed, = ctx.saved_tensors
        p, number, site = ctx.rule
        dx = _run(dy, p, number if seed is None else seed, site, None) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def _as_rows(t):
    """[rows, last dimension] with whatever strides the tensor has (a copy
    only where its leading dimensions cannot be one)."""
    return t.reshape(-1, t.shape[-1]) if t.dim() else t.reshape(1, 1)


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
    Differentiable once in ``x`` and ``residual``."""
    _block.check_tensor("x", x, tuple(_block.DTYPES))
    if residual is not None:
        _block.check_tensor("residual", residual, (x.dtype,), x.device)
        _block.require(residual.shape == x.shape, f"residual is {tuple(residual.shape)}, x {tuple(x.shape)}")
    _block.fill_rule(_block.GfDropoutRule(), p, seed, site, x.device)
    if x.numel() == 0:
        return x.clone() if residual is None else residual + x
    y = _Dropout.apply(_as_rows(x), None if residual is None else _as_rows(residual), p, seed, site)
    return y.view(x.shape)
