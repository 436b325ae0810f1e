"""The block operators inside torch's autograd machinery: checkpointing,
offloaded saved tensors."""
from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from guass_b200 import _block
from guass_b200.dropout import dropout
from guass_b200.feedforward import gated_feed_forward

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_timeouts():
    yield
    assert _block.device_flags() == 0


def inputs(rows=70, d=32, f=48):
    g = torch.Generator().manual_seed(3)
    x, w_in, w_out = (torch.randn(*s, generator=g).bfloat16().cuda() for s in ((rows, d), (2 * f, d), (d, f)))
    return x.requires_grad_(), (w_in * d ** -0.5).requires_grad_(), (w_out * f ** -0.5).requires_grad_()


def block(x, w_in, w_out, base):
    """Both dropouts from a seed that exists inside alone."""
    seed = base + 7
    y = gated_feed_forward(x, w_in, w_out, dropout_p=0.3, seed=seed, site=1)
    return dropout(y, 0.3, seed, site=2, residual=x)


@pytest.mark.parametrize("hooks", ["checkpoint", "reentrant", "save_on_cpu"])
def test_gradients_under_hooks_equal_the_plain_ones(hooks):
    leaves = inputs()
    base = torch.tensor([5], device="cuda")
    dy = torch.randn(70, 32, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()

    def gradients(forward):
        for t in leaves:
            t.grad = None
        y = forward()
        # memory of the size of a seed is taken and overwritten, as a program that goes on would
        junk = [torch.full((1,), 1 << 40, device="cuda") for _ in range(64)]
        y.backward(dy)
        del junk
        return [y.detach()] + [t.grad for t in leaves]

    want = gradients(lambda: block(*leaves, base))
    if hooks == "save_on_cpu":
        def forward():
            with torch.autograd.graph.save_on_cpu(pin_memory=True):
                return block(*leaves, base)
    else:
        def forward():
            return checkpoint(block, *leaves, base, use_reentrant=hooks == "reentrant")
    assert all(torch.equal(a, b) for a, b in zip(gradients(forward), want))


@pytest.mark.parametrize("hooks", ["checkpoint", "save_on_cpu"])
def test_a_changed_seed_is_refused_under_hooks(hooks):
    x, w_in, w_out = inputs()
    for fn in (lambda s: dropout(x, 0.5, s), lambda s: gated_feed_forward(x, w_in, w_out, dropout_p=0.5, seed=s)):
        seed = torch.tensor([1], device="cuda")
        if hooks == "checkpoint":
            y = checkpoint(fn, seed, use_reentrant=False)
        else:
            with torch.autograd.graph.save_on_cpu():
                y = fn(seed)
        seed.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_flag_watch_and_trainer_on_the_gpu():
    """A training step with the fused feed-forward looks at the flags without finding one; the copy is asynchronous."""
    from guass_b200 import sd15
    from guass_b200.adapters import BatchedAdapters

    cfg = sd15.tiny_config()
    cfg.feed_forward = "kernel"
    torch.manual_seed(0)
    with torch.device("cuda"):
        model = sd15.SD15UNet(cfg, dtype=torch.bfloat16)
    model.cuda()
    bank = BatchedAdapters(model.adapters(), out_dtype=torch.bfloat16)
    bank.install()
    tr = sd15.DataParallelTrainer(model, bank)
    inp = sd15.synthetic_inputs(cfg, 2, 1, device="cuda")
    tr._flags.flags.fill_(-1)  # overwritten by a copy of the device's zero
    tr._flags.look()
    torch.cuda.synchronize()
    assert tr._flags.flags.item() == 0
    for _ in range(3):
        assert torch.isfinite(tr.step(inp)).item()
    assert _block.device_flags() == 0
    tr._flags.flags.fill_(_block.GF_FLAG_TIMEOUT)
    with pytest.raises(RuntimeError, match="not valid"):
        tr.step(inp)
