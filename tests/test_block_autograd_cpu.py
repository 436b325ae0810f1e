"""The block operators' autograd functions on the CPU, their launches replaced
by recorders: what they keep for the backward and what they refuse."""
from __future__ import annotations

import ctypes
import gc
import weakref

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint

from guass_b200 import _block
from guass_b200 import dropout as dropout_module
from guass_b200 import feedforward as ff_module
from guass_b200 import int8 as int8_module


def seed_behind(rule) -> int:
    return ctypes.c_int64.from_address(rule.seed_ptr).value if rule.seed_ptr else rule.seed


@pytest.fixture
def launches(monkeypatch):
    """Lets CPU tensors through; every launch appends (kind, seed it would read)."""
    seen, alive = [], []

    def drop(x, rule, residual):
        assert all(ref() is not None for ref in alive), "the seed's memory is gone"
        seen.append(("dropout", seed_behind(rule)))
        return x * 2 if residual is None else x * 2 + residual

    def forward(x, w_in, w_out, b_in, b_out, activation, rule, keep):
        seen.append(("forward", seed_behind(rule)))
        return x * 2, (x.clone() if keep else None)

    def run(device, size_fn, fn, desc, *args, **kw):
        assert all(ref() is not None for ref in alive), "the seed's memory is gone"
        seen.append(("backward", seed_behind(desc.dropout)))

    monkeypatch.setattr(_block, "check_tensor", lambda *a: None)
    monkeypatch.setattr(dropout_module, "_run", drop)
    monkeypatch.setattr(ff_module, "_forward", forward)
    monkeypatch.setattr(_block, "run", run)
    return seen, alive


def operators():
    w_in, w_out = torch.ones(16, 4), torch.ones(4, 8)
    return {"dropout": lambda x, seed: dropout_module.dropout(x, 0.5, seed),
            "feed_forward": lambda x, seed: ff_module.gated_feed_forward(x, w_in, w_out, dropout_p=0.5, seed=seed)}


@pytest.mark.parametrize("op", ["dropout", "feed_forward"])
@pytest.mark.parametrize("hooks", ["none", "checkpoint", "save_on_cpu", "clone"])
def test_a_seed_made_on_the_way_lives_until_the_backward(launches, op, hooks):
    seen, alive = launches
    fn, base = operators()[op], torch.tensor([5])
    x = torch.ones(3, 4, requires_grad=True)

    def part(x):
        seed = base + 7
        if not alive:
            alive.append(weakref.ref(seed))
        return fn(x, seed)

    if hooks == "checkpoint":
        y = checkpoint(part, x, use_reentrant=False)
    elif hooks == "save_on_cpu":
        with torch.autograd.graph.save_on_cpu():
            y = part(x)
    elif hooks == "clone":  # what is packed is not the tensor itself, as when it is offloaded
        with torch.autograd.graph.saved_tensors_hooks(torch.clone, lambda t: t):
            y = part(x)
    else:
        y = part(x)
    gc.collect()
    y.sum().backward()
    assert {seed for _, seed in seen} == {12} and len(seen) >= 2


@pytest.mark.parametrize("op", ["dropout", "feed_forward"])
@pytest.mark.parametrize("hooks", ["none", "checkpoint", "clone"])
def test_a_seed_that_changed_is_refused(launches, op, hooks):
    fn, seed = operators()[op], torch.tensor([5])
    x = torch.ones(3, 4, requires_grad=True)
    if hooks == "checkpoint":
        y = checkpoint(lambda x: fn(x, seed), x, use_reentrant=False)
    elif hooks == "clone":
        with torch.autograd.graph.saved_tensors_hooks(torch.clone, lambda t: t):
            y = fn(x, seed)
    else:
        y = fn(x, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(launches, grad):
    """A tangent is refused, not dropped, wherever it comes in; primals work in a dual level as outside."""
    drop, ff = dropout_module.dropout, ff_module.gated_feed_forward
    x, w_in, w_out, b_in, b_out = (torch.ones(*s) for s in ((3, 4), (16, 4), (4, 8), (16,), (4,)))
    q, s = torch.ones(4, 4, dtype=torch.int8), torch.ones(4)
    seen, _ = launches
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        calls = [lambda: drop(dual(x), 0.5, 1), lambda: drop(x, 0.5, 1, residual=dual(x)),
                 lambda: int8_module.int8_linear(dual(x), q, s), lambda: int8_module.int8_linear(x, q, dual(s)),
                 lambda: int8_module.int8_matmul(q, dual(s), q, s),
                 lambda: int8_module.int8_matmul(q, s, q, s, bias=dual(b_out.bfloat16()))]
        args = [x, w_in, w_out, b_in, b_out]
        calls += [lambda i=i: ff(*args[:i], dual(args[i]), *args[i + 1:]) for i in range(5)]
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert not seen
        drop(x, 0.5, 1), ff(*args)
    assert len(seen) == 2


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(),
                                  lambda m: m.to("cpu", torch.float16)])
def test_casting_a_model_keeps_8_bit_scales(launches, cast):
    scale = torch.tensor([1.0 + 2.0 ** -20, 0.3])
    layer = int8_module.Int8Linear(torch.ones(2, 16, dtype=torch.int8), scale, torch.zeros(2))
    model = cast(torch.nn.Sequential(layer))
    assert model[0] is layer and layer.weight_scale.dtype == torch.float32
    assert torch.equal(layer.weight_scale, scale) and layer.q_weight.dtype == torch.int8
    assert torch.equal(layer.state_dict()["weight_scale"], scale) and layer.bias.dtype != torch.float32


@pytest.mark.parametrize("op", ["dropout", "feed_forward"])
def test_a_seed_whose_memory_moved_is_read_where_it_is(launches, op):
    """An assignment to .data gives the seed other memory: the backward reads that, never the old address."""
    seen, _ = launches
    seed = torch.tensor([5])
    x = torch.ones(3, 4, requires_grad=True)
    y = operators()[op](x, seed)
    seed.data = torch.tensor([5])
    gc.collect()
    y.sum().backward()
    assert seen[-1][1] == 5


def test_a_seed_that_left_its_device_is_refused():
    kept = _block.KeptRule(_block.GfDropoutRule(), torch.tensor([5]))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        kept.get(torch.device("cuda", 0))
