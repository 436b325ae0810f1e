"""The block operators where the framework calls them: the SD1.5-shaped UNet's
feed-forward and dropout in adapter training, merged projections in 8 bits."""
from __future__ import annotations

import pytest
import torch

import block_reference as ref
from guass_b200 import _block, sd15
from guass_b200.adapters import BatchedAdapters

pytestmark = pytest.mark.gpu


def setup(dtype=torch.bfloat16, **kw):
    cfg = sd15.tiny_config()
    for k, v in kw.items():
        setattr(cfg, k, v)
    torch.manual_seed(0)
    with torch.device("cuda"):
        model = sd15.SD15UNet(cfg, dtype=dtype)
    model.cuda()
    bank = BatchedAdapters(model.adapters(), out_dtype=dtype, fused_weight=True)
    bank.install()
    return model, bank, sd15.DataParallelTrainer(model, bank, seed=3)


def inputs(seed=2):
    return sd15.synthetic_inputs(sd15.tiny_config(), 2, seed, device="cuda")


@pytest.mark.parametrize("p", [0.0, 0.2])
def test_block_feed_forward_modes(p):
    """Both modes of one block against the 64-bit form: the kernels within
    their bound; the composed operations within it and their own extra
    roundings (u, the activation and the product in bf16: three half steps of
    every hidden term, and as many again of what they feed)."""
    model, _, _ = setup(feed_forward="kernel", dropout=p)
    blk = next(m for m in model.modules() if isinstance(m, sd15.TransformerBlock))
    x = torch.randn(2, 64, 32, device="cuda").bfloat16().requires_grad_()
    dy = torch.randn(2, 64, 32, device="cuda").bfloat16()
    seed = torch.tensor([9], device="cuda") if p else None
    keep = ref.keep_mask(128, 128, p, 9, blk.site + 2) / (1 - p) if p else None
    flat = x.detach().view(128, 32)
    want = ref.feed_forward(flat, blk.ff_in.weight, blk.ff_out.weight, blk.ff_in.bias, blk.ff_out.bias, "gelu", keep,
                            dy.view(128, 32), torch.bfloat16)
    for fused in (True, False):
        blk.fused_ff = fused
        y = blk.feed_forward(x, seed)
        dx, = torch.autograd.grad(y, [x], dy)
        for got, (value, bound) in ((y, want["y"]), (dx, want["dx"])):
            err = (got.detach().double().cpu().view(128, 32) - value).abs()
            assert (err / (bound if fused else 6 * bound)).max() <= 1.0


@pytest.mark.parametrize("mode", ["kernel", "composed"])
@pytest.mark.parametrize("p", [0.0, 0.1])
def test_training_steps(mode, p):
    model, bank, tr = setup(feed_forward=mode, dropout=p)
    for _ in range(2):
        loss = tr.step(inputs())
    assert torch.isfinite(loss).item() and bank.batch.device_flags() == 0 and _block.device_flags() == 0
    assert (model.dropout_seed is None) if p == 0 else model.dropout_seed.item() == 5  # 3, advanced twice
    first = tr.backward(inputs())
    grads = [q.grad.clone() for q in tr.params]
    for q in tr.params:
        assert torch.isfinite(q.grad).all() and q.grad.abs().sum() > 0
        q.grad = None
    again = tr.backward(inputs())  # the same seed: the same masks, so the same loss
    torch.testing.assert_close(again, first, rtol=1e-3, atol=0)
    if p:
        model.eval()
        with torch.no_grad():
            still = sd15.diffusion_loss(model, inputs(), tr.alphas_cumprod)
            model.dropout_seed.add_(1)
            assert torch.equal(sd15.diffusion_loss(model, inputs(), tr.alphas_cumprod), still)  # none in eval mode
        model.train()
        with torch.no_grad():
            assert not torch.equal(sd15.diffusion_loss(model, inputs(), tr.alphas_cumprod), still)
    assert len(grads) == len(tr.params)


def test_dropouts_have_their_own_sites():
    model, _, _ = setup(dropout=0.1)
    sites = [m.site + i for m in model.modules() if isinstance(m, sd15.TransformerBlock) for i in range(3)]
    assert len(set(sites)) == len(sites) > 3


@pytest.mark.parametrize("fused", [False, True])
def test_merged_layers_in_8_bits(fused):
    torch.manual_seed(0)
    with torch.device("cuda"):
        model = sd15.SD15UNet(sd15.tiny_config(), dtype=torch.bfloat16)
    model.cuda()
    bank = BatchedAdapters(model.adapters(), out_dtype=torch.bfloat16, fused_weight=fused)
    bank.install()
    deltas = [d.detach().float() for d in bank.render()]
    m, d = bank.modules[0], deltas[0]
    x = torch.randn(2, 5, m.in_features, device="cuda").bfloat16()
    inp = inputs()
    with torch.no_grad():
        before, whole = m(x), model(inp.latents, inp.t, inp.text)
        bank.quantize_merged()
        with pytest.raises(RuntimeError, match="already"):
            bank.quantize_merged()
        after, whole8 = m(x), model(inp.latents, inp.t, inp.text)
        qx, sx = ref.quantise(x.view(10, -1))
        qw, sw = ref.quantise(d if fused else m.weight.float() + d)
        want = (qx.double() @ qw.double().t()) * sx.double()[:, None] * sw.double()
        want = want + (0 if m.bias is None else m.bias.double().cpu())
        err = (after.double().cpu().view(10, -1) - want).abs()
        assert (err <= ref.rounding(want, torch.bfloat16) + 2.0 ** -20 * want.abs().max()).all()
        assert torch.isfinite(whole8).all() and not torch.equal(whole8, whole)
        bank.unquantize()
        assert torch.equal(m(x), before)
        assert not any("forward" in q.__dict__ for q in bank.modules) or fused


def test_model_renderer_serves_8_bits():
    """quantize_merged under ModelRenderer: no render per forward; uninstalling leaves 8-bit serving."""
    from guass_b200.adapters import ModelRenderer

    torch.manual_seed(0)
    with torch.device("cuda"):
        model = sd15.SD15UNet(sd15.tiny_config(), dtype=torch.bfloat16)
    model.cuda()
    r = ModelRenderer(model, fused_weight=True, out_dtype=torch.bfloat16)
    inp = inputs()
    with torch.no_grad():
        before = model(inp.latents, inp.t, inp.text)
        r.bank.quantize_merged()
        r.bank._current = None  # a render would set it
        a = model(inp.latents, inp.t, inp.text)
        assert r.bank._current is None and torch.equal(a, model(inp.latents, inp.t, inp.text))
        assert torch.isfinite(a).all() and not torch.equal(a, before)
        r.bank.unquantize()
        assert torch.equal(model(inp.latents, inp.t, inp.text), before)
        r.bank.quantize_merged()
        r.remove()
    assert not any("forward" in m.__dict__ for m in model.adapters().values())


def test_8_bits_refuse_training():
    torch.manual_seed(0)
    with torch.device("cuda"):
        model = sd15.SD15UNet(sd15.tiny_config(), dtype=torch.bfloat16)
    model.cuda()
    bank = BatchedAdapters(model.adapters(), out_dtype=torch.bfloat16)
    bank.install()
    bank.render()
    bank.quantize_merged()
    m = bank.modules[0]
    x = torch.randn(3, m.in_features, device="cuda").bfloat16().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        m(x)
    with torch.no_grad():
        assert m(x).shape == (3, m.out_features)


def test_8_bits_after_merging_count_the_delta_once():
    torch.manual_seed(0)
    with torch.device("cuda"):
        model = sd15.SD15UNet(sd15.tiny_config(), dtype=torch.bfloat16)
    model.cuda()
    bank = BatchedAdapters(model.adapters(), out_dtype=torch.bfloat16)
    bank.install()
    m = bank.modules[0]
    bank.merge_into_weights()
    merged = m.weight.detach().float()
    bank.quantize_merged()
    q, scale = ref.quantise(merged)
    layer = bank._int8[0][2]
    assert torch.equal(layer.q_weight.cpu(), q) and torch.equal(layer.weight_scale.cpu(), scale)
    bank.unquantize()
    bank.unmerge_weights()
