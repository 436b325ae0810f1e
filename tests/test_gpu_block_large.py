"""The feed-forward where element offsets pass 2^31."""
from __future__ import annotations

import pytest
import torch

import block_reference as ref
from guass_b200 import _block
from guass_b200.feedforward import gated_feed_forward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out", [24, 21])  # results through TMA stores, and element by element
def test_offsets_past_2_31(out):
    """h and the gradient of u hold more than 2^31 elements.  Rows repeat with a period, and a row's results depend on
    that row alone: every period equals the first, which is held to the 64-bit form."""
    period, d, f = 1000, 16, 4096
    count = 540  # 540000 x 4096 = 2.2e9 elements of h, twice that of du
    g = torch.Generator().manual_seed(7)
    rows = torch.randn(period, d, generator=g).bfloat16()
    dys = torch.randn(period, out, generator=g).bfloat16()
    w_in = (torch.randn(2 * f, d, generator=g) * d ** -0.5).bfloat16()
    w_out = (torch.randn(out, f, generator=g) * f ** -0.5).bfloat16()
    x = rows.cuda().repeat(count, 1).requires_grad_()
    y = gated_feed_forward(x, w_in.cuda(), w_out.cuda())
    dx, = torch.autograd.grad(y, [x], dys.cuda().repeat(count, 1))
    want = ref.feed_forward(rows, w_in, w_out, None, None, "gelu", None, dys, torch.bfloat16)
    for got, (value, bound) in ((y.detach(), want["y"]), (dx, want["dx"])):
        got = got.view(count, period, -1)
        assert ((got[0].double().cpu() - value).abs() <= bound).all()
        assert torch.equal(got, got[:1].expand_as(got))
    assert _block.device_flags() == 0
