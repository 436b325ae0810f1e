"""Gated feed-forward block (GEGLU / SwiGLU) in hand-written kernels.

``y = h w_out^T + b_out`` with ``h = dropout(value * act(gate))`` and
``value, gate = (x w_in^T + b_in).chunk(2, -1)``: the feed-forward of a
transformer block, e.g. of :class:`guass_b200.sd15.TransformerBlock`.  Both
input projections, the activation, the product and the dropout are one kernel;
the output projection is a second.  Matrices are bf16 or fp16, products
accumulate in fp32.

The backward computes the projections and the dropout mask again from the
block's input, so that a training forward keeps the input alone (and the
hidden activations where ``w_out`` is trained).  It computes only the gradients
that are asked for: with frozen weights (how the Gaussian adapters are
trained) that is two kernels.
"""
from __future__ import annotations

import torch

from guass_b200 import _block

_TYPES = (torch.bfloat16, torch.float16)


def _describe(x, w_in, w_out, b_in, b_out, activation, rule):
    f = _block.GfGatedFf()
    f.tokens, f.in_features = x.shape
    f.out_features, f.hidden = w_out.shape
    f.dtype = _block.DTYPES[x.dtype]
    f.activation = _block.ACTIVATIONS[activation]
    f.dropout = rule
    f.x, f.ld_x = x.data_ptr(), _block.ld(x)
    f.w_in, f.ld_w_in = w_in.data_ptr(), _block.ld(w_in)
    f.w_out, f.ld_w_out = w_out.data_ptr(), _block.ld(w_out)
    if b_in is not None:
        f.b_in = b_in.data_ptr()
    if b_out is not None:
        f.b_out = b_out.data_ptr()
    return f


def _forward(x, w_in, w_out, b_in, b_out, activation, rule, keep):
    """(y, h): h is the saved state, None without ``keep``."""
    L = _block.lib()
    d, (out, hidden) = x.shape[-1], w_out.shape
    shape = x.shape
    x, w_in, w_out = _block.rows_of(x, d), _block.rows_of(w_in, d), _block.rows_of(w_out, hidden)
    b_in, b_out = (None if b is None else b.contiguous() for b in (b_in, b_out))
    f = _describe(x, w_in, w_out, b_in, b_out, activation, rule)
    y = torch.empty(*shape[:-1], out, dtype=x.dtype, device=x.device)
    f.y, f.ld_y = y.data_ptr(), out
    hp = -(-hidden // 64) * 64
    h, use_room = None, None
    if keep:
        h = torch.empty(f.tokens, hp, dtype=x.dtype, device=x.device)
        f.h = h.data_ptr()
    else:
        def use_room(pointer):
            f.h = pointer
    if f.tokens:
        _block.run(x.device, L.gf_gated_ff_workspace_bytes, L.gf_gated_ff_forward, f, query=(0,),
                   room=0 if keep else 2 * f.tokens * hp, use_room=use_room)
    return y, h


class _GatedFeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, w_out, b_in, b_out, activation, p, seed, site):
        need = ctx.needs_input_grad
        rule = _block.make_rule(p, seed, site, x.device)
        y, h = _forward(x, w_in, w_out, b_in, b_out, activation, rule, need[2])
        ctx.save_for_backward(x, w_in, w_out, b_in, h)
        ctx.activation, ctx.kept = activation, _block.KeptRule(rule, seed)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w_in, w_out, b_in, h = ctx.saved_tensors
        need, (out, hidden), d, shape = ctx.needs_input_grad, w_out.shape, w_in.shape[1], x.shape
        dy, x = _block.rows_of(dy, out), _block.rows_of(x, d)
        w_in, w_out = _block.rows_of(w_in, d), _block.rows_of(w_out, hidden)
        b_in = None if b_in is None else b_in.contiguous()
        L = _block.lib()
        f = _describe(x, w_in, w_out, b_in, None, ctx.activation, ctx.kept.get(dy.device))
        f.dy, f.ld_dy = dy.data_ptr(), _block.ld(dy)
        if h is not None:
            f.h = h.data_ptr()

        def grad(wanted, *shape):
            return torch.empty(shape, dtype=dy.dtype, device=dy.device) if wanted else None

        dx, dw_in, dw_out = grad(need[0], *shape), grad(need[1], 2 * hidden, d), grad(need[2], out, hidden)
        db_in, db_out = grad(need[3], 2 * hidden), grad(need[4], out)
        for name, g in (("dx", dx), ("dw_in", dw_in), ("dw_out", dw_out), ("db_in", db_in), ("db_out", db_out)):
            if g is not None:
                setattr(f, name, g.data_ptr())
        _block.run(dy.device, L.gf_gated_ff_workspace_bytes, L.gf_gated_ff_backward, f, query=(1,))
        return dx, dw_in, dw_out, db_in, db_out, None, None, None, None


def _check(x, w_in, w_out, b_in, b_out, activation) -> None:
    _block.check_tensor("x", x, _TYPES)
    device, dtypes = x.device, (x.dtype,)
    _block.check_tensor("w_in", w_in, dtypes, device)
    _block.check_tensor("w_out", w_out, dtypes, device)
    if x.dim() < 1 or w_in.dim() != 2 or w_out.dim() != 2:
        raise ValueError("x needs a feature dimension, w_in and w_out two dimensions")
    d, (out, hidden), (rows, cols) = x.shape[-1], w_out.shape, w_in.shape
    if rows != 2 * hidden or cols != d:
        raise ValueError(f"w_in is {(rows, cols)}, expected {(2 * hidden, d)} for x {tuple(x.shape)} and w_out "
                         f"{(out, hidden)}")
    if d == 0 or hidden == 0 or out == 0:
        raise ValueError("feature sizes must be positive")
    for name, b, n in (("b_in", b_in, rows), ("b_out", b_out, out)):
        if b is not None:
            _block.check_tensor(name, b, dtypes, device)
            if b.dim() != 1 or b.shape[0] != n:
                raise ValueError(f"{name} must be [{n}], got {tuple(b.shape)}")
    if activation not in _block.ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_block.ACTIVATIONS)}, got {activation!r}")


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

    Differentiable once in every tensor, in reverse mode.  Work goes to the current stream of
    ``x``'s device; nothing synchronises, and both passes can be captured."""
    _check(x, w_in, w_out, b_in, b_out, activation)
    _block.refuse_tangents("gated_feed_forward", x, w_in, w_out, b_in, b_out)
    if torch.is_grad_enabled() and (x.requires_grad or w_in.requires_grad or w_out.requires_grad
                                    or b_in is not None and b_in.requires_grad
                                    or b_out is not None and b_out.requires_grad):
        return _GatedFeedForward.apply(x, w_in, w_out, b_in, b_out, activation, dropout_p, seed, site)
    rule = _block.make_rule(dropout_p, seed, site, x.device)
    return _forward(x, w_in, w_out, b_in, b_out, activation, rule, False)[0]
