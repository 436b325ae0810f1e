"""Gated feed-forward block (GEGLU / SwiGLU) in hand-written kernels.

``y = h w_out^T + b_out`` with ``h = dropout(value * act(gate))`` and
``value, gate = (x w_in^T + b_in).chunk(2, -1)``: the feed-forward of a
transformer block, e.g. of :class:`guass_b200.sd15.TransformerBlock`.  Both
input projections, the activation, the product and the dropout are one kernel;
the output projection is a second.  Matrices are bf16 or fp16, products
accumulate in fp32.

The training forward saves, in the room the two projections would take, what
the backward multiplies with: the activation and its slope times the value,
each with the dropout folded in.  The backward computes only the gradients that are asked for: with frozen weights (how
the Gaussian adapters are trained) that is two kernels.
"""
from __future__ import annotations

import ctypes

import torch

from guass_b200 import _block, _lib

_TYPES = (torch.bfloat16, torch.float16)


def _describe(x, w_in, w_out, b_in, b_out, activation, p, seed, site):
    f = _block.GfGatedFf()
    f.tokens, f.in_features = x.shape
    f.hidden, f.out_features = w_out.shape[1], w_out.shape[0]
    f.dtype = _block.DTYPES[x.dtype]
    f.activation = _block.ACTIVATIONS[activation]
    _block.fill_rule(f.dropout, p, seed, site, x.device)
    f.x, f.ld_x = x.data_ptr(), _block.ld(x)
    f.w_in, f.ld_w_in = w_in.data_ptr(), _block.ld(w_in)
    f.w_out, f.ld_w_out = w_out.data_ptr(), _block.ld(w_out)
    f.b_in = b_in.data_ptr() if b_in is not None else None
    f.b_out = b_out.data_ptr() if b_out is not None else None
    return f


def _launch(L, f, backward: bool, device) -> None:
    n = L.gf_gated_ff_workspace_bytes(ctypes.byref(f), int(backward))
    if n == 0:
        raise _lib.GfieldError(_lib.GF_ERR_INVALID_ARG, _lib.last_error())
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    fn = L.gf_gated_ff_backward if backward else L.gf_gated_ff_forward
    _lib.check(fn(ctypes.byref(f), ws.data_ptr(), n, torch.cuda.current_stream(device).cuda_stream))


def _forward(x, w_in, w_out, b_in, b_out, activation, p, seed, site, keep):
    L = _block.lib()
    f = _describe(x, w_in, w_out, b_in, b_out, activation, p, seed, site)
    hp = -(-f.hidden // 64) * 64
    y = torch.empty(f.tokens, f.out_features, dtype=x.dtype, device=x.device)
    h = torch.empty(f.tokens, hp, dtype=x.dtype, device=x.device)
    u = torch.empty(f.tokens, 2 * hp, dtype=x.dtype, device=x.device) if keep else None
    f.y, f.ld_y, f.h = y.data_ptr(), f.out_features, h.data_ptr()
    f.u = u.data_ptr() if keep else None
    if f.tokens:
        _launch(L, f, False, x.device)
    return y, h, u


class _GatedFeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, w_out, b_in, b_out, activation, p, seed, site):
        with _block.on_device(x):
            y, h, u = _forward(x, w_in, w_out, b_in, b_out, activation, p, seed, site, True)
        wants_w_out = ctx.needs_input_grad[2]
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, w_in, w_out, u, h if wants_w_out else None,
                              seed if isinstance(seed, torch.Tensor) else None)
        ctx.rule = (activation, p, None if isinstance(seed, torch.Tensor) else seed, site)
        ctx.shape = x.shape
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w_in, w_out, u, h, seed = ctx.saved_tensors
        activation, p, number, site = ctx.rule
        need = ctx.needs_input_grad
        dy = _block.rows_of(dy, w_out.shape[0])
        with _block.on_device(dy):
            L = _block.lib()
            stand_in = x if x is not None else dy.new_empty(0, ctx.shape[1])
            f = _describe(stand_in, w_in, w_out, None, None, activation, p, number if seed is None else seed, site)
            f.tokens = ctx.shape[0]
            f.u = u.data_ptr()
            f.h = h.data_ptr() if h is not None else None
            f.dy, f.ld_dy = dy.data_ptr(), _block.ld(dy)

            def grad(wanted, *shape):
                return torch.empty(*shape, dtype=dy.dtype, device=dy.device) if wanted else None

            dx = grad(need[0], f.tokens, f.in_features)
            dw_in = grad(need[1], 2 * f.hidden, f.in_features)
            dw_out = grad(need[2], f.out_features, f.hidden)
            db_in = grad(need[3], 2 * f.hidden)
            db_out = grad(need[4], f.out_features)
            for name, g in (("dx", dx), ("dw_in", dw_in), ("dw_out", dw_out), ("db_in", db_in), ("db_out", db_out)):
                setattr(f, name, g.data_ptr() if g is not None else None)
            _launch(L, f, True, dy.device)
        return dx, dw_in, dw_out, db_in, db_out, None, None, None, None


def gated_feed_forward(x, w_in, w_out, b_in=None, b_out=None, *, activation: str = "gelu", dropout_p: float = 0.0,
                       seed=0, site: int = 0):
    """``linear(dropout(value * act(gate)), w_out, b_out)`` where
    ``value, gate = linear(x, w_in, b_in).chunk(2, -1)``.

    ``x`` [..., in], ``w_in`` [2 * hidden, in] (value rows first), ``w_out``
    [out, hidden], biases [2 * hidden] and [out] or None; all bf16 or all fp16
    on one CUDA device, of any sizes and strides (operands whose rows do not
    start on 16-byte boundaries cost a copy).  ``activation``: ``"gelu"`` (the
    error-function form) or ``"silu"``.  ``dropout_p``, ``seed`` and ``site``
    drop hidden activations by the rule of :func:`guass_b200.dropout.dropout`
    on the hidden ``[rows, hidden]``; a seed tensor must not change between
    the forward and its backward.  Returns [..., out].

    Differentiable once in every tensor.  Work goes to the current stream of
    ``x``'s device; nothing synchronises, and both passes can be captured."""
    _block.check_tensor("x", x, _TYPES)
    for name, t in (("w_in", w_in), ("w_out", w_out), ("b_in", b_in), ("b_out", b_out)):
        if t is not None or name[0] == "w":
            _block.check_tensor(name, t, (x.dtype,), x.device)
    _block.require(x.dim() >= 1 and w_in.dim() == 2 and w_out.dim() == 2, "x needs a feature dimension, w_in and "
                   "w_out two dimensions")
    d, hidden = x.shape[-1], w_out.shape[1]
    _block.require(w_in.shape[0] == 2 * hidden and w_in.shape[1] == d,
                   f"w_in is {tuple(w_in.shape)}, expected {(2 * hidden, d)} for x {tuple(x.shape)} and w_out "
                   f"{tuple(w_out.shape)}")
    _block.require(min(d, hidden, w_out.shape[0]) > 0, "feature sizes must be positive")
    _block.require(b_in is None or tuple(b_in.shape) == (2 * hidden,), "b_in must be [2 * hidden]")
    _block.require(b_out is None or tuple(b_out.shape) == (w_out.shape[0],), "b_out must be [out]")
    _block.require(activation in _block.ACTIVATIONS,
                   f"activation must be one of {sorted(_block.ACTIVATIONS)}, got {activation!r}")
    _block.fill_rule(_block.GfDropoutRule(), dropout_p, seed, site, x.device)
    flat, wi, wo = _block.rows_of(x, d), _block.rows_of(w_in, d), _block.rows_of(w_out, hidden)
    bi, bo = (b.contiguous() if b is not None else None for b in (b_in, b_out))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (flat, wi, wo, bi, bo)):
        y = _GatedFeedForward.apply(flat, wi, wo, bi, bo, activation, dropout_p, seed, site)
    else:
        with _block.on_device(x):
            y = _forward(flat, wi, wo, bi, bo, activation, dropout_p, seed, site, False)[0]
    return y.view(*x.shape[:-1], w_out.shape[0])
