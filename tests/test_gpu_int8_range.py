"""The 8-bit product at the ends of fp32's range: results that fit are finite."""
from __future__ import annotations

import pytest
import torch

import block_reference as ref
from guass_b200 import _block
from guass_b200.int8 import int8_linear, int8_matmul, quantize_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("big,small", [(1e36, 1e-9), (-2e30, 1e-3), (2.0 ** 96, 2.0 ** -40), (3e38, 1e-38), (1e-38, 3e38)])
def test_large_scales(big, small, dtype):
    """A sum times its row's scale would pass 2^128; the product of all three does not."""
    m, n, k = 70, 96, 1280
    g = torch.Generator().manual_seed(5)
    a, b = (torch.randint(-127, 128, (r, k), generator=g, dtype=torch.int8) for r in (m, n))
    a[3], b[5] = 127, 127  # the largest sum of these
    sa, sb = torch.rand(m, generator=g) + 0.5, torch.rand(n, generator=g) + 0.5
    # beside rows of ordinary scale, where those times a large `small` would not be past the range themselves
    sa[::2 if small < 1 else 1] *= big / 1.5
    sb *= small / 1.5
    got = int8_matmul(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), out_dtype=dtype).double().cpu()
    want = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()
    assert want.abs().max() < torch.finfo(dtype).max
    # the sum's conversion and two products in fp32, each normal or subnormal, and the store
    bound = 3 * 2.0 ** -24 * want.abs() + 2.0 ** -149 + ref.rounding(want, dtype)
    assert torch.isfinite(got).all() and ((got - want).abs() <= 1.02 * bound).all()
    assert _block.device_flags() == 0


def test_rows_near_the_end_of_the_range():
    """Activations near fp32's largest value against small weights."""
    g = torch.Generator().manual_seed(6)
    x = torch.randn(40, 512, generator=g).clamp(-3, 3) / 3 * 3e38
    w = torch.randn(64, 512, generator=g) * 1e-6
    qw, sw = quantize_rows(w.cuda())
    y = int8_linear(x.cuda(), qw, sw).double().cpu()
    qx, sx = ref.quantise(x)
    want = (qx.double() @ qw.cpu().double().t()) * sx.double()[:, None] * sw.cpu().double()
    assert torch.isfinite(y).all()
    assert ((y - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all()


def test_nan_scales_stay_nan_beside_large_ones():
    a = torch.ones(3, 32, dtype=torch.int8, device="cuda")
    sa = torch.tensor([float("nan"), 1e37, 1.0], device="cuda")
    sb = torch.tensor([1e-7, float("nan")], device="cuda")
    y = int8_matmul(a, sa, a[:2], sb, out_dtype=torch.float32).cpu()
    assert torch.equal(torch.isnan(y), torch.tensor([[True, True], [False, True], [False, True]]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [300, 700, 1300])
@pytest.mark.parametrize("cols", [333, 512, 1280, 1288, 1536, 1537, 2048, 2056])
def test_quantised_rows_in_every_variant(rows, cols, dtype):
    """A warp or a CTA for a row, held or read twice: the same numbers, those of the definition."""
    x = (torch.randn(rows, cols, generator=torch.Generator().manual_seed(cols)) * 3).to(dtype)
    x[0], x[rows - 1, cols - 1], x[rows // 2, 0] = 0, float("nan"), float("inf")
    q, scale = quantize_rows(x.cuda())
    want, ws = ref.quantise(x)
    assert torch.equal(q.cpu(), want) and torch.equal(scale.cpu().nan_to_num(nan=-1.0), ws.nan_to_num(nan=-1.0))
