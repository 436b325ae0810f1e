"""The gate's activations element by element, far out on both sides: value 1
and gate x through identity weights, so that the output is act(x) rounded to
the type and the input's gradient its slope."""
from __future__ import annotations

import pytest
import torch

import block_reference as ref
from guass_b200 import _block
from guass_b200.feedforward import gated_feed_forward

pytestmark = pytest.mark.gpu

N = 64
# relative error of an activation and of a slope's two terms in fp32: 2.2e-5 at most (see the kernel), 2^-15 = 3.1e-5
RELATIVE = 2.0 ** -15


def gates(dtype, low, high, rows):
    """[rows, N] gates of ``dtype``, evenly spread, zero and the smallest steps around it among them."""
    g = torch.linspace(low, high, rows * N, dtype=torch.float64)
    g[: N // 2] = torch.linspace(-1, 1, N // 2, dtype=torch.float64) * 2.0 ** -10
    g[0] = 0
    return g.to(dtype).view(rows, N)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("rows", [4, 8, 300])  # the walk over the weights, and the product kernel
@pytest.mark.parametrize("low,high", [(-13, -3), (-8, -3), (-3, 3), (3, 13)])
def test_activation_and_slope(low, high, rows, act, dtype):
    x = gates(dtype, low, high, rows).cuda().requires_grad_()
    eye = torch.eye(N, dtype=dtype, device="cuda")
    w_in = torch.cat([torch.zeros_like(eye), eye])
    b_in = torch.cat([torch.ones(N, dtype=dtype), torch.zeros(N, dtype=dtype)]).cuda()
    y = gated_feed_forward(x, w_in, eye, b_in, activation=act)
    g = x.detach().double().cpu()
    value, slope, _ = ref.activation(act, g)
    err = (y.detach().double().cpu() - value).abs()
    assert (err <= RELATIVE * value.abs() + (1 + RELATIVE) * ref.rounding(value, dtype)).all(), \
        (err / value.abs()).nan_to_num(0).max()
    dx, = torch.autograd.grad(y, [x], torch.ones_like(y))
    # the slope is a sum whose terms may cancel: Phi + g phi, or sig + g sig (1 - sig)
    terms = slope.abs() + 2 * torch.minimum(value.abs() / g.abs().clamp_min(1e-30), (slope - value / g).abs().nan_to_num(0))
    err = (dx.double().cpu() - slope).abs()
    assert (err <= RELATIVE * terms + (1 + RELATIVE) * ref.rounding(slope, dtype)).all()
    assert _block.device_flags() == 0
