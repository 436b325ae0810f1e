"""Dropout at positions past 32 bits, and in a training step whose gradients
must follow the seed."""
from __future__ import annotations

import pytest
import torch

import block_reference as ref
from guass_b200 import sd15
from guass_b200.adapters import BatchedAdapters
from guass_b200.dropout import dropout

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["rows of one vector", "one element", "rows next to each other"])
def test_positions_past_32_bits(layout):
    """rows x groups of 2^31 and more (8 columns a group in aligned rows, else 4), small inputs read through strides."""
    p, seed, site = 0.5, 17, 1
    if layout == "rows of one vector":
        rows, cols = (1 << 20) + 1, 1 << 14
        x = torch.full((1, cols), 2.0, dtype=torch.bfloat16, device="cuda").expand(rows, cols)
    elif layout == "one element":
        rows, cols = (1 << 21) + 1, 1 << 12
        x = torch.full((1, 1), 2.0, dtype=torch.bfloat16, device="cuda").expand(rows, cols)
    else:
        rows, cols = (1 << 20) + 1, (1 << 13) + 3
        x = torch.full((rows + 2 * cols,), 2.0, dtype=torch.bfloat16, device="cuda").as_strided((rows, cols), (1, 2))
    y = dropout(x, p, seed, site=site)
    for r in (0, 1, rows // 2, rows - 2, rows - 1):
        for c in (0, cols - 256):
            words = [ref.philox([(c + j) // 4, r, site, 0], [seed, 0])[(c + j) % 4] for j in range(256)]
            keep = torch.tensor([w >= 1 << 31 for w in words])
            assert torch.equal(y[r, c:c + 256].cpu(), torch.where(keep, 4.0, 0.0).bfloat16()), (r, c)
    del y
    torch.cuda.empty_cache()


def test_gradients_follow_the_seed():
    """Two backwards with one seed draw the same masks: their gradients differ by flipped roundings alone (one bf16
    step, 2^-8, at each of some hundred tensors in a row: at most 2^-8 * sqrt(100) ~ 2^-5 of their norm).  Another
    seed changes them by more."""
    cfg = sd15.tiny_config()
    cfg.feed_forward, cfg.dropout = "kernel", 0.2
    torch.manual_seed(0)
    with torch.device("cuda"):
        model = sd15.SD15UNet(cfg, dtype=torch.bfloat16)
    model.cuda()
    bank = BatchedAdapters(model.adapters(), out_dtype=torch.bfloat16, fused_weight=True)
    bank.install()
    tr = sd15.DataParallelTrainer(model, bank, seed=3)
    inp = sd15.synthetic_inputs(cfg, 2, 2, device="cuda")

    def gradients(seed):
        with torch.no_grad():
            model.dropout_seed.fill_(seed)
        tr.backward(inp)
        flat = torch.cat([q.grad.flatten().double() for q in tr.params])
        for q in tr.params:
            q.grad = None
        return flat

    first, again, other = gradients(3), gradients(3), gradients(4)
    same, changed = ((first - g).norm() / first.norm() for g in (again, other))
    assert same <= 2.0 ** -5 < changed
