"""DataParallelTrainer and the seed of a model's dropout, on the CPU."""
from __future__ import annotations

import ctypes

import pytest
import torch
from torch import nn

from guass_b200 import sd15
from guass_b200.adapters import BatchedAdapters
from oracle_batch import OracleBatch


class OtherModel(nn.Module):
    """A model of someone else: adapters, no dropout and no seed of one."""

    def __init__(self):
        super().__init__()
        torch.manual_seed(0)
        self.unet = sd15.SD15UNet(sd15.tiny_config(), dtype=torch.float32)

    def adapters(self):
        return self.unet.adapters()

    def forward(self, x, t, ctx):
        return self.unet(x, t, ctx)


def trainer(model, **kw):
    bank = BatchedAdapters(model.adapters(), batch_factory=OracleBatch, out_dtype=torch.float32)
    bank.install()
    return sd15.DataParallelTrainer(model, bank, **kw)


def test_any_model_with_adapters_trains():
    tr = trainer(OtherModel())
    before = tr.params[0].detach().clone()
    loss = tr.step(sd15.synthetic_inputs(sd15.tiny_config(), 1, 3, dtype=torch.float32))
    assert torch.isfinite(loss) and not torch.equal(tr.params[0], before)


def test_a_resumed_run_goes_on_with_its_masks(monkeypatch):
    """seed + n draws after a resume what the run would have drawn from step n on."""
    seeds = []

    def dropout(x, p, seed, *, site=0, residual=None):
        seeds.append((int(seed), site))
        return x if residual is None else residual + x

    monkeypatch.setattr(sd15, "dropout", dropout)

    def run(start, steps):
        cfg = sd15.tiny_config()
        cfg.dropout = 0.1
        torch.manual_seed(0)
        tr = trainer(sd15.SD15UNet(cfg, dtype=torch.float32), seed=start)
        seeds.clear()
        for _ in range(steps):
            tr.step(sd15.synthetic_inputs(cfg, 1, 3, dtype=torch.float32))
        return list(seeds)

    whole = run(7, 3)
    assert len(set(whole)) == len(whole)  # no mask twice
    assert whole[2 * len(whole) // 3:] == run(7 + 2, 1)


def test_a_wait_that_ran_out_stops_the_training(monkeypatch):
    """The fused feed-forward's condition bits, copied behind a step, end the next one."""
    from guass_b200 import _block

    class Library:  # sets what the device would have set during the second step
        calls = 0

        def gf_block_status_async(self, pointer, stream):
            Library.calls += 1
            ctypes.c_uint32.from_address(pointer).value = _block.GF_FLAG_TIMEOUT if Library.calls == 2 else 0
            return 0

    plain = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *a, pin_memory=False, **kw: plain(*a, **kw))
    monkeypatch.setattr(_block, "lib", Library)
    monkeypatch.setattr(_block, "call", lambda device, fn, *args: fn(*args, None))
    model = OtherModel()
    tr = trainer(model)
    assert tr._flags is None  # composed feed-forwards, and no GPU
    tr._flags = _block.FlagWatch(torch.device("cpu"))
    inputs = sd15.synthetic_inputs(sd15.tiny_config(), 1, 3, dtype=torch.float32)
    tr.step(inputs)
    tr.step(inputs)
    with pytest.raises(RuntimeError, match="0x10"):
        tr.step(inputs)
    assert Library.calls == 2


def test_a_model_need_not_be_a_module():
    class Plain:
        def __init__(self, model):
            self.model, self.adapters = model, model.adapters

        def __call__(self, *args):
            return self.model(*args)

    tr = trainer(Plain(OtherModel()))
    assert torch.isfinite(tr.step(sd15.synthetic_inputs(sd15.tiny_config(), 1, 3, dtype=torch.float32)))
