"""8-bit serving of merged adapters (guass_b200.adapters) on the CPU: which
weight is quantised and whose forward serves when.  The layer is a test double
that keeps its weight; the GPU tests cover the product."""
from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F
from torch import nn

from guass_b200 import int8
from guass_b200.adapters import BatchedAdapters, ModelRenderer
from oracle_batch import OracleBatch
from test_adapters import FakeLinear


class KeptLinear(nn.Module):
    def __init__(self, weight, bias):
        super().__init__()
        self.weight, self.bias = weight.detach().clone(), bias

    @classmethod
    def from_weight(cls, weight, bias=None):
        return cls(weight, bias)

    def forward(self, x):
        return F.linear(x, self.weight, self.bias)


class Layer(FakeLinear):
    def forward(self, x):
        return F.linear(x, self.weight + self.compute_delta_weight(), self.bias)

    def compute_delta_weight(self):  # without a binding: no adapter
        return torch.zeros_like(self.weight)


@pytest.fixture(autouse=True)
def kept_layers(monkeypatch):
    monkeypatch.setattr(int8, "Int8Linear", KeptLinear)


def modules():
    return {"a": Layer(40, 70, 6, 1, scale=0.5), "b": Layer(33, 40, 4, 3, scale=0.5)}


def make(fused=False):
    mods = modules()
    bank = BatchedAdapters(mods, batch_factory=OracleBatch, out_dtype=torch.float32, fused_weight=fused)
    base = [m.weight.detach().clone() for m in bank.modules]
    with torch.no_grad():
        full = [d.clone() if fused else w + d for w, d in zip(base, bank.render())]
    bank._current = None
    return bank, full


def served(bank):
    return [layer.weight for _, _, layer in bank._int8]


@pytest.mark.parametrize("between", ["nothing", "render", "unfreeze"])
def test_quantising_after_merging_counts_the_delta_once(between):
    bank, full = make()
    bank.install()
    bank.merge_into_weights()
    if between == "render":
        bank.render()
    elif between == "unfreeze":
        bank.unfreeze()
    bank.quantize_merged()
    for got, m, want in zip(served(bank), bank.modules, full):
        assert torch.equal(got, m.weight) and torch.allclose(got, want, rtol=0, atol=1e-6)


@pytest.mark.parametrize("again", ["render", "hook", "unfreeze"])
def test_merged_weights_serve_the_delta_once(again):
    """A render after merge_into_weights (ModelRenderer renders before every forward) adds nothing."""
    bank, full = make()
    model = nn.ModuleDict(zip("ab", bank.modules))
    bank.install()
    bank.merge_into_weights()
    if again == "hook":
        r = ModelRenderer.__new__(ModelRenderer)
        r.bank = bank
        r._before_forward(model, ())
    elif again == "unfreeze":
        bank.unfreeze()
        bank.render()
    else:
        bank.render()
    for m, want in zip(bank.modules, full):
        x = torch.ones(2, m.in_features)
        assert torch.allclose(m(x), F.linear(x, want), rtol=0, atol=1e-4)
    bank.unmerge_weights()
    with torch.no_grad():
        for m, d, want in zip(bank.modules, bank.render(), full):
            assert torch.allclose(m.weight + d, want, rtol=0, atol=1e-6)


def test_merging_twice_and_freezing_merged_weights_are_refused():
    bank, full = make()
    bank.freeze()
    bank.merge_into_weights()
    with pytest.raises(RuntimeError, match="already"):
        bank.merge_into_weights()
    with pytest.raises(RuntimeError, match="unmerge_weights"):
        bank.freeze()
    bank.unmerge_weights()
    for m, d, want in zip(bank.modules, bank.render(), full):  # frozen before the merge, so frozen still
        assert torch.equal(m.compute_delta_weight(), d) and torch.allclose(m.weight + d, want, rtol=0, atol=1e-6)
    bank.unfreeze()


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("own_forward", [False, True])
@pytest.mark.parametrize("order", ["install first", "quantise first"])
def test_installing_and_quantising_in_any_order(order, fused, own_forward):
    """8 bits serve from quantize_merged until unquantize or uninstall, which leave the modules as they were."""
    bank, full = make(fused)
    plain = [m.forward for m in bank.modules]
    if own_forward:  # a forward that someone else put on the module
        for m, f in zip(bank.modules, plain):
            m.forward = lambda x, f=f: f(x) + 1
    before = [m.__dict__.get("forward") for m in bank.modules]
    x = [torch.ones(2, m.in_features) for m in bank.modules]

    def eight_bits():
        return all(torch.equal(m(v), F.linear(v, w)) for m, v, w in zip(bank.modules, x, full))

    if order == "install first":
        bank.install()
        bank.quantize_merged()
    else:
        bank.quantize_merged()
        bank.install()
    assert eight_bits()
    bank.install()  # again: nothing changes
    assert eight_bits()
    bank.unquantize()
    with torch.no_grad():
        bank.render()
        for m, v, w in zip(bank.modules, x, full):
            want = F.linear(v, w) + (1 if own_forward and not fused else 0)
            assert torch.allclose(m(v), want, rtol=0, atol=1e-4)
    bank.quantize_merged()
    assert eight_bits()
    bank.uninstall()
    assert [m.__dict__.get("forward") for m in bank.modules] == before and not bank._int8
    assert all("compute_delta_weight" not in m.__dict__ or m.compute_delta_weight().eq(0).all() for m in bank.modules)


def test_a_layer_that_cannot_be_quantised_changes_nothing(monkeypatch):
    bank, full = make()
    bank.install()
    calls = []

    def from_weight(weight, bias=None):
        calls.append(weight)
        if len(calls) == 2:
            raise MemoryError
        return KeptLinear(weight, bias)

    with monkeypatch.context() as m:
        m.setattr(KeptLinear, "from_weight", from_weight)
        with pytest.raises(MemoryError):
            bank.quantize_merged()
    assert not bank._int8 and not any("forward" in m.__dict__ for m in bank.modules)
    bank.quantize_merged()
    assert all(torch.equal(a, b) for a, b in zip(served(bank), full))


@pytest.mark.parametrize("installed", [False, True])
def test_a_new_k_ends_serving_the_old_one(installed):
    bank, _ = make()
    if installed:
        bank.install()
    bank.quantize_merged()
    m = bank.modules[0]
    for name in ("mu_raw", "chol_raw", "amp"):
        setattr(m, name, nn.Parameter(getattr(m, name).detach()[:-1]))
    assert bank.shapes_changed()
    fresh = bank.rebuilt()
    assert not bank._int8 and not fresh._int8 and not any("forward" in q.__dict__ for q in bank.modules)
    fresh.quantize_merged()
    with torch.no_grad():
        assert all(torch.equal(w, q.weight + d) for w, q, d in zip(served(fresh), fresh.modules, fresh.render()))
    fresh.uninstall()
    assert not any("forward" in q.__dict__ for q in bank.modules)
