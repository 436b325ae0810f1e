"""The block operators on the GPU against their 64-bit definitions: gated
feed-forward (forward, every gradient), dropout, the 8-bit product."""
from __future__ import annotations

import pytest
import torch

import block_reference as ref
from guass_b200 import _block
from guass_b200.dropout import dropout
from guass_b200.feedforward import gated_feed_forward
from guass_b200.int8 import Int8Linear, int8_linear, int8_matmul, quantize_rows

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def no_timeouts():
    yield
    assert _block.device_flags() == 0


def normal(*shape, seed, dtype, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).cuda()


def check(got, want, name=""):
    value, bound = want
    err = (got.detach().double().cpu() - value).abs()
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert worst <= 1.0, f"{name}: {worst:.2f} times the bound"


# ---------------------------------------------------------------------------
# feed-forward

def ff_inputs(m, d, f, o, dtype, bias, seed=0):
    t = dict(x=normal(m, d, seed=seed, dtype=dtype), w_in=normal(2 * f, d, seed=seed + 1, dtype=dtype, std=d ** -0.5),
             w_out=normal(o, f, seed=seed + 2, dtype=dtype, std=f ** -0.5), b_in=None, b_out=None)
    if bias:
        t.update(b_in=normal(2 * f, seed=seed + 3, dtype=dtype, std=0.3), b_out=normal(o, seed=seed + 4, dtype=dtype))
    return t


def ff_check(t, act, p=0.0, seed=0, site=0, wants=("x", "w_in", "w_out", "b_in", "b_out")):
    """Runs forward and backward and compares everything that was asked for."""
    leaves = {n: t[n].detach().requires_grad_() for n in wants if t[n] is not None}
    args = {**t, **leaves}
    y = gated_feed_forward(args["x"], args["w_in"], args["w_out"], args["b_in"], args["b_out"], activation=act,
                           dropout_p=p, seed=seed, site=site)
    m, f, dtype = t["x"].shape[0], t["w_out"].shape[1], t["x"].dtype
    number = int(seed.item()) if isinstance(seed, torch.Tensor) else seed
    keep = ref.keep_mask(m, f, p, number, site) / (1 - p) if p else None
    dy = normal(*y.shape, seed=77, dtype=dtype) if leaves else None
    want = ref.feed_forward(t["x"], t["w_in"], t["w_out"], t["b_in"], t["b_out"], act, keep, dy, dtype)
    check(y, want["y"], "y")
    if leaves:
        for n, g in zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)):
            check(g, want["d" + n], "d" + n)


FF_SIZES = [
    # tokens, in, hidden, out
    (1, 64, 64, 64),
    (1, 320, 1280, 320),
    (2, 8, 16, 24),          # one k step, mostly padding
    (3, 1, 1, 1),            # smallest features
    (7, 5, 3, 9),            # nothing aligned
    (64, 640, 192, 136),
    (127, 72, 130, 61),
    (128, 320, 1280, 320),
    (129, 333, 1001, 77),    # past one row tile, odd everywhere
    (300, 1280, 640, 1280),  # long sums: K ranges
    (1000, 96, 448, 200),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("size", FF_SIZES)
def test_ff_forward_and_gradients(size, dtype):
    act = "gelu" if sum(size) % 2 else "silu"
    ff_check(ff_inputs(*size, dtype, bias=size[0] % 2 == 1), act)


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("p", [0.0, 0.25])
def test_ff_variants(act, bias, p):
    ff_check(ff_inputs(200, 136, 264, 104, BF16, bias), act, p=p, seed=12345678901234, site=7)


@pytest.mark.parametrize("wants", [(), ("x",), ("w_in",), ("w_out",), ("b_in",), ("b_out",), ("x", "w_out"),
                                   ("w_in", "b_out")])
def test_ff_wanted_gradients_only(wants):
    ff_check(ff_inputs(70, 48, 80, 56, BF16, True), "gelu", p=0.1, seed=3, wants=wants)


def test_ff_many_tiles_per_cta():
    """More output tiles than CTAs: both accumulators, several rounds of the pipeline."""
    t = ff_inputs(4096 + 40, 64, 1280, 64, BF16, True)
    ff_check(t, "gelu", p=0.1, seed=9, wants=("x", "w_in"))


def test_ff_large_gates():
    """Gates far out on both tails, where the activation is 0 or the identity."""
    t = ff_inputs(64, 64, 128, 64, BF16, False)
    t["x"] = t["x"] * 20
    ff_check(t, "gelu")
    ff_check(t, "silu")


@pytest.mark.parametrize("off", [0, 1, 4])
def test_ff_strided_operands(off):
    """Column slices of wider matrices (aligned and not), a transposed weight and a transposed dy."""
    base = ff_inputs(90, 80, 96, 72, FP16, True)
    wide = {n: normal(base[n].shape[0], base[n].shape[1] + 24, seed=50 + i, dtype=FP16) for i, n in
            enumerate(("x", "w_in", "w_out"))}
    t = dict(base)
    for n, w in wide.items():
        w[:, off:off + base[n].shape[1]] = base[n]
        t[n] = w[:, off:off + base[n].shape[1]]
    t["w_out"] = t["w_out"].t().contiguous().t()
    t["b_in"] = torch.cat([t["b_in"][:1], t["b_in"]])[1:]  # a bias that starts off the 16-byte grid
    ff_check(t, "gelu")
    x = t["x"].detach().requires_grad_()
    y = gated_feed_forward(x, t["w_in"], t["w_out"], t["b_in"], t["b_out"])
    dy = normal(72, 90, seed=5, dtype=FP16).t()
    a, = torch.autograd.grad(y, [x], dy, retain_graph=True)
    b, = torch.autograd.grad(y, [x], dy.contiguous())
    assert torch.equal(a, b)
    s, = torch.autograd.grad(gated_feed_forward(x, t["w_in"], t["w_out"], t["b_in"], t["b_out"]).sum(), [x])
    one, = torch.autograd.grad(gated_feed_forward(x, t["w_in"], t["w_out"], t["b_in"], t["b_out"]), [x],
                               torch.ones_like(y))
    assert torch.equal(s, one)  # an expanded dy (stride 0)


def test_ff_shapes_and_empty():
    t = ff_inputs(24, 64, 128, 40, BF16, True)
    y = gated_feed_forward(*(t[n] for n in ("x", "w_in", "w_out", "b_in", "b_out")))
    z = gated_feed_forward(t["x"].view(2, 3, 4, 64), *(t[n] for n in ("w_in", "w_out", "b_in", "b_out")))
    assert z.shape == (2, 3, 4, 40) and torch.equal(z.view(24, 40), y)
    v = gated_feed_forward(t["x"][0], *(t[n] for n in ("w_in", "w_out", "b_in", "b_out")))
    assert v.shape == (40,)
    leaves = [t[n].detach().requires_grad_() for n in ("w_in", "w_out", "b_in", "b_out")]
    e = gated_feed_forward(t["x"][:0].view(0, 5, 64), *leaves)
    assert e.shape == (0, 5, 40)
    for g in torch.autograd.grad(e, leaves, torch.empty_like(e)):
        assert not g.any()


def test_ff_rows_do_not_mix():
    """A row of infinities or NaN reaches its own output and input gradient only."""
    t = ff_inputs(150, 72, 100, 48, BF16, True)
    dy = normal(150, 48, seed=8, dtype=BF16)

    def run(x, dy):
        x = x.detach().requires_grad_()
        y = gated_feed_forward(x, t["w_in"], t["w_out"], t["b_in"], t["b_out"])
        return y.detach(), torch.autograd.grad(y, [x], dy)[0]

    clean = run(t["x"], dy)
    for bad in (float("inf"), float("nan")):
        x, g = t["x"].clone(), dy.clone()
        x[3], g[140, 5] = bad, bad
        dirty = run(x, g)
        rows = torch.arange(150, device="cuda")
        assert torch.equal(clean[0][rows != 3], dirty[0][rows != 3]) and not torch.isfinite(dirty[0][3]).any()
        ok = (rows != 3) & (rows != 140)
        assert torch.equal(clean[1][ok], dirty[1][ok]) and not torch.isfinite(dirty[1][140]).any()


def test_ff_is_reproducible():
    t = ff_inputs(700, 320, 640, 320, BF16, True)
    leaves = [t[n].requires_grad_() for n in ("x", "w_in", "w_out", "b_in", "b_out")]
    dy = normal(700, 320, seed=1, dtype=BF16)
    runs = []
    for _ in range(2):
        y = gated_feed_forward(*leaves, dropout_p=0.1, seed=5)
        runs.append([y, *torch.autograd.grad(y, leaves, dy)])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_ff_gradient_by_differences():
    """The slope of the loss along a direction, from two forwards, against the gradient."""
    t = ff_inputs(40, 64, 96, 32, FP16, True)
    x = t["x"].detach().requires_grad_()
    args = [t[n] for n in ("w_in", "w_out", "b_in", "b_out")]
    dy = normal(40, 32, seed=4, dtype=FP16)
    grad, = torch.autograd.grad(gated_feed_forward(x, *args, dropout_p=0.2, seed=1), [x], dy)
    step = (normal(40, 64, seed=6, dtype=FP16) * 2 ** -4).to(FP16)
    hi, lo = (t["x"] + step), (t["x"] - step)  # fp16 sums: take the exact difference below
    loss = [(gated_feed_forward(v, *args, dropout_p=0.2, seed=1).double() * dy.double()).sum() for v in (hi, lo)]
    along = (grad.double() * (hi.double() - lo.double())).sum()
    # each y is off by at most ~4 half steps of fp16 of its terms (|y| ~ 1, 1280 of them, random signs:
    # 5 standard deviations), the second-order terms cancel and the third are |step|^3 ~ 2e-4 of them
    noise = 5 * (1280 ** 0.5) * 4 * 2 ** -11 * 2 ** 0.5
    assert abs((loss[0] - loss[1] - along).item()) <= noise + 0.02 * along.abs().item()


# ---------------------------------------------------------------------------
# dropout

DROP_SIZES = [(1, 1), (1, 3), (5, 4), (77, 768), (33, 1001), (1000, 7), (3, 4096), (257, 40)]


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("size", DROP_SIZES)
@pytest.mark.parametrize("with_residual", [False, True])
def test_dropout_values_and_gradients(size, dtype, with_residual):
    p, seed, site = 0.3, 0x123456789ABCDEF, 0xFFFFFFFF
    x = normal(*size, seed=1, dtype=dtype).requires_grad_()
    r = normal(*size, seed=2, dtype=dtype).requires_grad_() if with_residual else None
    y = dropout(x, p, seed, site=site, residual=r)
    keep = ref.keep_mask(*size, p, seed, site)
    part = x.detach().double().cpu() * keep / (1 - p)
    want = part + (r.detach().double().cpu() if with_residual else 0)
    # scale and product round in fp32, the sum and the store once more each
    check(y, (want, 3 * 2.0 ** -24 * (part.abs() + want.abs()) + ref.rounding(want, dtype)), "y")
    assert y.is_contiguous()
    dy = normal(*size, seed=3, dtype=dtype)
    grads = torch.autograd.grad(y, [x] + ([r] if with_residual else []), dy)
    g = dy.double().cpu() * keep / (1 - p)
    check(grads[0], (g, 3 * 2.0 ** -24 * g.abs() + ref.rounding(g, dtype)), "dx")
    assert bool(((grads[0].cpu() == 0) | keep).all())
    if with_residual:
        assert torch.equal(grads[1], dy)


@pytest.mark.parametrize("p", [0.0, 1e-9, 0.1, 0.5, 0.999])
def test_dropout_rate(p):
    n = 1 << 20
    y = dropout(torch.ones(1024, 1024, device="cuda"), p, 7)
    dropped = int((y == 0).sum())
    assert abs(dropped - p * n) <= 6 * (n * p * (1 - p)) ** 0.5 + 1e-3
    assert torch.equal(y[y != 0], torch.full_like(y[y != 0], 1 / (1 - p)))


def test_dropout_layouts_agree():
    """The same mask for any strides: transposed, sliced (aligned or not), expanded, more dimensions."""
    x = normal(48, 96, seed=3, dtype=BF16)
    want = dropout(x, 0.4, 11)
    wide = torch.zeros(48, 200, dtype=BF16, device="cuda")
    for off in (0, 1, 8):
        wide[:, off:off + 96] = x
        assert torch.equal(dropout(wide[:, off:off + 96], 0.4, 11), want)
        assert torch.equal(dropout(x, 0.4, 11, residual=wide[:, off:off + 96]), dropout(x, 0.4, 11, residual=x))
    assert torch.equal(dropout(x.t().contiguous().t(), 0.4, 11), want)
    assert torch.equal(dropout(x.view(4, 12, 96), 0.4, 11).view(48, 96), want)
    four = x.view(4, 12, 8, 12).permute(1, 0, 3, 2)
    assert torch.equal(dropout(four, 0.4, 11), dropout(four.contiguous(), 0.4, 11))
    row = x[:1].expand(48, 96)
    assert torch.equal(dropout(row, 0.4, 11), dropout(row.contiguous(), 0.4, 11))
    assert torch.equal(dropout(x.flip(0), 0.4, 11), dropout(x.flip(0).contiguous(), 0.4, 11))
    assert torch.equal(dropout(x[0], 0.4, 11), want[0])
    assert dropout(x[:0], 0.4, 11).shape == (0, 96)
    assert torch.equal(dropout(x, 0.4, torch.tensor([11], device="cuda")), want)
    assert not torch.equal(dropout(x, 0.4, 11, site=1), want) and not torch.equal(dropout(x, 0.4, 12), want)


def test_dropout_drops_whatever_was_there():
    x = torch.full((64, 64), float("nan"), device="cuda")
    y = dropout(x, 0.5, 1)
    keep = ref.keep_mask(64, 64, 0.5, 1, 0).cuda()
    assert torch.equal(torch.isnan(y), keep) and not y[~keep].any()
    same = torch.ones(8, 8, device="cuda").requires_grad_()
    z = dropout(same, 0.5, 1, residual=same)  # one tensor in both places
    g, = torch.autograd.grad(z.sum(), [same])
    assert torch.equal(g, z.detach())


def test_ff_and_dropout_share_the_rule():
    """The block with dropout on its hidden activations equals an identity-free
    composition: hidden mask of (seed, site) over [rows, hidden]."""
    t = ff_inputs(40, 32, 64, 64, FP16, False)
    eye = torch.eye(64, dtype=FP16, device="cuda")
    h = gated_feed_forward(t["x"], t["w_in"], eye)
    d = gated_feed_forward(t["x"], t["w_in"], eye, dropout_p=0.5, seed=21, site=4)
    assert torch.equal(d, dropout(h, 0.5, 21, site=4))  # 1 / (1 - p) = 2: no rounding


@pytest.mark.parametrize("tokens", [6, 200])
def test_ff_drops_whatever_was_there(tokens):
    """One hidden unit that is infinite for every row reaches only the rows that keep it, forward and backward."""
    t = ff_inputs(tokens, 32, 64, 40, BF16, True)
    clean = {n: t[n].detach().clone() for n in t}
    t["b_in"][5] = float("inf")
    kept = ref.keep_mask(tokens, 64, 0.5, 9, 0)[:, 5].cuda()
    assert kept.any() and not kept.all()
    out = []
    for v in (clean, t):
        x = v["x"].detach().requires_grad_()
        y = gated_feed_forward(x, v["w_in"], v["w_out"], v["b_in"], v["b_out"], dropout_p=0.5, seed=9)
        out.append((y.detach(), torch.autograd.grad(y, [x], torch.ones_like(y))[0]))
    for a, b in zip(*out):
        assert torch.equal(a[~kept], b[~kept])
    assert not torch.isfinite(out[1][0][kept]).any()


# ---------------------------------------------------------------------------
# 8-bit product

@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("size", [(1, 1), (1, 16), (3, 5), (4, 1280), (231, 333), (40, 2048), (9, 2056), (5, 5001)])
def test_quantize_rows(size, dtype):
    x = normal(*size, seed=4, dtype=dtype, std=3.0)
    if size[0] > 2:
        x[1] = 0
        x[2, 0] = float("inf")
        if size[0] > 3:
            x[3, -1] = float("nan")
    q, scale = quantize_rows(x)
    want, ws = ref.quantise(x)
    assert torch.equal(q.cpu(), want) and torch.equal(scale.cpu().nan_to_num(nan=-1.0), ws.nan_to_num(nan=-1.0))
    assert q.stride(0) % 16 == 0 and q.untyped_storage().nbytes() == q.shape[0] * q.stride(0)
    wide = torch.zeros(size[0], size[1] + 3, dtype=dtype, device="cuda")
    wide[:, 1:1 + size[1]] = x
    assert torch.equal(quantize_rows(wide[:, 1:1 + size[1]])[0], q)


def test_quantize_tiny_rows():
    x = torch.tensor([[2.0 ** -101, 0], [2.0 ** -99, -2.0 ** -100], [1e-42, 1e-42], [3e38, -1e38]], device="cuda")
    q, s = quantize_rows(x)
    want, ws = ref.quantise(x)
    assert torch.equal(q.cpu(), want) and torch.equal(s.cpu(), ws)


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("size", [(1, 1, 1), (1, 1280, 1280), (4, 320, 1280), (77, 640, 768), (231, 1001, 333),
                                  (128, 96, 128), (129, 33, 200), (700, 2561, 130), (20000, 320, 64)])
def test_int8_matmul(size, dtype):
    m, n, k = size
    g = torch.Generator().manual_seed(m + n + k)
    a, b = (torch.randint(-128, 128, (r, k), generator=g, dtype=torch.int8) for r in (m, n))
    sa, sb = torch.rand(m, generator=g) * 0.1, torch.rand(n, generator=g) * 0.1
    bias = torch.randn(n, generator=g).to(dtype) if n % 2 else None
    got = int8_matmul(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), None if bias is None else bias.cuda(), out_dtype=dtype)
    acc = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()
    want = acc + (0 if bias is None else bias.double())
    # the sum is exact; converted, scaled twice and added in fp32, stored once
    check(got, (want, 4 * 2.0 ** -24 * (acc.abs() + want.abs()) + ref.rounding(want, dtype)))


def test_int8_longest_sum():
    """K = 131071 of the most negative values: 2^31 - 2^14, the largest sum that is still exact."""
    k = 131071
    a = torch.full((2, k), -128, dtype=torch.int8, device="cuda")
    one = torch.ones(2, device="cuda")
    got = int8_matmul(a, one, a, one, out_dtype=FP32)
    assert torch.equal(got.cpu(), torch.full((2, 2), float(k * 16384)))


@pytest.mark.parametrize("off", [0, 1, 16])
def test_int8_strided_operands(off):
    g = torch.Generator().manual_seed(1)
    a, b = (torch.randint(-127, 128, (r, 160), generator=g, dtype=torch.int8).cuda() for r in (50, 60))
    sa, sb = torch.rand(50, device="cuda"), torch.rand(120, device="cuda")[::2]
    x, w = a[:, off:off + 100], b[:, off:off + 100]
    want = int8_matmul(x.contiguous(), sa, w.contiguous(), sb.contiguous())
    assert torch.equal(int8_matmul(x, sa, w, sb), want)
    assert torch.equal(int8_matmul(x.t().contiguous().t(), sa, w, sb), want)


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("lead", [(), (1,), (0,), (4, 77)])
def test_int8_linear(lead, dtype):
    w, bias = normal(96, 200, seed=1, dtype=dtype, std=0.1), normal(96, seed=2, dtype=dtype)
    x = normal(*lead, 200, seed=3, dtype=dtype)
    layer = Int8Linear.from_weight(w, bias)
    y = layer(x)
    assert y.shape == (*lead, 96) and y.dtype == dtype
    qx, sx = ref.quantise(x.reshape(-1, 200))
    qw, sw = ref.quantise(w)
    acc = (qx.double() @ qw.double().t()) * sx.double()[:, None] * sw.double()
    want = acc + bias.double().cpu()
    check(y.view(-1, 96), (want, 4 * 2.0 ** -24 * (acc.abs() + want.abs()) + ref.rounding(want, dtype)))
    assert int8_linear(x, layer.q_weight, layer.weight_scale, out_dtype=FP32).dtype == FP32


def test_int8_rows_do_not_mix():
    layer = Int8Linear.from_weight(normal(40, 64, seed=1, dtype=BF16))
    x = normal(140, 64, seed=2, dtype=BF16)
    clean = layer(x)
    x[5, 3], x[131, 0] = float("nan"), float("-inf")
    dirty = layer(x)
    rows = torch.arange(140, device="cuda")
    ok = (rows != 5) & (rows != 131)
    assert torch.equal(clean[ok], dirty[ok]) and torch.isnan(dirty[~ok]).all()


# ---------------------------------------------------------------------------
# streams, graphs, several calls at once

def test_other_streams_and_overlap():
    t = ff_inputs(500, 320, 640, 320, BF16, True)
    args = [t[n] for n in ("x", "w_in", "w_out", "b_in", "b_out")]
    layer = Int8Linear.from_weight(t["w_in"])
    want = gated_feed_forward(*args, dropout_p=0.1, seed=2), layer(t["x"]), dropout(t["x"], 0.1, 2)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((gated_feed_forward(*args, dropout_p=0.1, seed=2), layer(t["x"]), dropout(t["x"], 0.1, 2)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_captured_step_sees_new_seeds():
    """A block as a training step uses it, captured once: dropout on the hidden
    activations and on the branch, forward and backward; replays with another
    seed and other inputs equal eager runs with them."""
    t = ff_inputs(300, 64, 256, 64, BF16, True)
    x = t["x"].detach().requires_grad_()
    w = [t[n] for n in ("w_in", "w_out", "b_in", "b_out")]
    seed = torch.tensor([5], dtype=torch.int64, device="cuda")
    dy = normal(300, 64, seed=9, dtype=BF16)

    def step():
        y = gated_feed_forward(x, *w, dropout_p=0.2, seed=seed, site=1)
        z = dropout(y, 0.2, seed, site=2, residual=x)
        grad, = torch.autograd.grad(z, [x], dy)
        return z.detach(), grad  # a graph of x that lives on would tie the next capture to its stream

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs with workspaces of their own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for value in (5, 6, -1):
        with torch.no_grad():
            seed.fill_(value)
            x.copy_(normal(300, 64, seed=value + 20, dtype=BF16))
        want = [v.detach().clone() for v in step()]
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_captured_int8():
    layer = Int8Linear.from_weight(normal(320, 333, seed=1, dtype=FP16))
    x = normal(9, 333, seed=2, dtype=FP16)
    layer(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = layer(x)
    x.copy_(normal(9, 333, seed=3, dtype=FP16))
    g.replay()
    assert torch.equal(y, layer(x))


def test_seed_changed_before_backward_is_refused():
    x = torch.ones(4, 4, device="cuda", requires_grad=True)
    t = ff_inputs(4, 8, 16, 8, BF16, False)
    leaf = t["x"].requires_grad_()
    seed = torch.tensor([1], device="cuda")
    made = dropout(x, 0.5, seed), gated_feed_forward(leaf, t["w_in"], t["w_out"], dropout_p=0.5, seed=seed)
    seed.add_(1)
    for y in made:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_no_second_derivative():
    x = torch.ones(4, 8, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(dropout(x, 0.5, 1).square().sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), [x])


def test_ff_long_sums_and_wide_rows():
    """K ranges joined in order (a long K and few tiles), rows past 2^16 columns."""
    ff_check(ff_inputs(16, 24, 33000, 40, BF16, True), "gelu", wants=("x", "w_out"))
    ff_check(ff_inputs(2100, 24, 40, 64, FP16, True), "silu")


def test_ff_one_input_in_two_blocks():
    """Two blocks in a row on the same input, whose gradient is the sum of both."""
    t, s = (ff_inputs(50, 32, 48, 32, FP16, True, seed=k) for k in (1, 20))
    x = t["x"].detach().requires_grad_()

    def block(w, v):
        return gated_feed_forward(v, *(w[n] for n in ("w_in", "w_out", "b_in", "b_out")), dropout_p=0.1, seed=2)

    dy = normal(50, 32, seed=3, dtype=FP16)
    both, = torch.autograd.grad([block(t, x), block(s, x)], [x], [dy, dy])
    one, = torch.autograd.grad(block(t, x), [x], dy)
    two, = torch.autograd.grad(block(s, x), [x], dy)
    assert torch.equal(both, one + two)


def test_dropout_large_positions():
    """Elements whose offset passes 2^31 (as bytes and as elements), few rows and many."""
    for rows, cols in ((3, 1 << 30), (1 << 20, 2100)):
        x = torch.ones(1, 1, dtype=BF16, device="cuda").expand(rows, cols)
        y = dropout(x, 0.5, 17, site=1)
        for r in (0, rows - 1):
            c = min(cols, 4096)
            mask = ref.keep_mask(1, 8, 0.5, 17, 1)  # row 0: the reference's own start
            words = [ref.philox([(cols - c + j) // 4, r, 1, 0], [17, 0])[(cols - c + j) % 4] >= 1 << 31 for j in range(c)]
            assert torch.equal(y[r, cols - c:].cpu() != 0, torch.tensor(words))
            if r == 0:
                assert torch.equal(y[0, :8].cpu() != 0, mask[0])
        del y


def test_int8_many_rows_past_2_31_bytes():
    """A result whose byte offsets pass 2^31."""
    m, n, k = 300_000, 4096, 32
    a = torch.ones(m, k, dtype=torch.int8, device="cuda")
    a[-1] = 3
    b = torch.ones(n, k, dtype=torch.int8, device="cuda")
    one = torch.ones(m, device="cuda")
    y = int8_matmul(a, one, b, one[:n])
    assert (y[:1000] == 32).all() and (y[-1] == 96).all() and (y[-1000:-1] == 32).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("size", [(320, 1280, 320), (2056, 72, 40), (77, 130, 9), (1280, 4100, 24)])
def test_ff_few_tokens(size, tokens, dtype):
    """The walk over the weights (up to 8 tokens) and its border, rows of any length on 16-byte boundaries."""
    d, f, o = size
    t = ff_inputs(tokens, d, f, o, dtype, bias=True)
    for n in ("x", "w_in", "w_out"):  # rows padded to whole 16 bytes, with values that must not be read as theirs
        rows, cols = t[n].shape
        wide = torch.full((rows, -(-cols // 8) * 8 + 8), float("nan"), dtype=dtype, device="cuda")
        wide[:, :cols] = t[n]
        t[n] = wide[:, :cols]
    ff_check(t, "gelu", p=0.25, seed=4, site=2)
    ff_check(t, "silu", wants=())


def test_refusals_on_the_gpu():
    t = ff_inputs(4, 8, 16, 8, BF16, True)
    x, wi, wo, bi, bo = (t[n] for n in ("x", "w_in", "w_out", "b_in", "b_out"))
    for args in ((x, wi[:-1], wo), (x, wi[:, 1:], wo), (x, wi, wo[:, :-1]), (x, wi, wo, bi[1:]), (x, wi, wo, bi, bo[1:]),
                 (x, wi, wo[:0]), (x[:, :0], wi[:, :0], wo), (x, wi[0], wo)):
        with pytest.raises(ValueError):
            gated_feed_forward(*args)
    for bad in (x.half(), x.float(), x.double()):
        with pytest.raises(TypeError):
            gated_feed_forward(bad, wi, wo)
    with pytest.raises(TypeError):
        gated_feed_forward(x, wi, wo, bi.float())
    with pytest.raises(ValueError, match="activation"):
        gated_feed_forward(x, wi, wo, activation="relu")
    for kw in (dict(dropout_p=1.0), dict(dropout_p=-0.1), dict(dropout_p=0.1, site=-1)):
        with pytest.raises(ValueError):
            gated_feed_forward(x, wi, wo, **kw)
        with pytest.raises(ValueError):
            gated_feed_forward(x.detach().requires_grad_(), wi, wo, **kw)
    with pytest.raises(TypeError):
        gated_feed_forward(x, wi, wo, dropout_p=0.1, seed=torch.ones(1, device="cuda"))
    with pytest.raises(ValueError):
        gated_feed_forward(x, wi, wo, dropout_p=0.1, seed=torch.ones(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(RuntimeError):
        gated_feed_forward(x, wi, wo, dropout_p=0.1, seed=torch.ones(1, dtype=torch.int64))
    with pytest.raises(RuntimeError):
        gated_feed_forward(x, wi.cpu(), wo)
    with pytest.raises(ValueError):
        dropout(x, 0.5, 1, residual=x[:2])
    with pytest.raises(TypeError):
        dropout(x, 0.5, 1, residual=x.float())
    with pytest.raises(TypeError):
        dropout(x.long(), 0.5, 1)
    q, s = quantize_rows(wi)
    for args in ((q[:, 1:], s, q, s), (q, s[1:], q, s), (q, s, q, s[1:]), (q, s, q[:0], s[:0]), (q[0], s, q, s)):
        with pytest.raises(ValueError):
            int8_matmul(*args)
    with pytest.raises(ValueError):
        int8_matmul(q, s, q, s, out_dtype=torch.float64)
    with pytest.raises(TypeError):
        int8_matmul(q, s, q, s, bias=torch.zeros(32, device="cuda"))
    with pytest.raises(TypeError):
        int8_matmul(q, s.double(), q, s)
    with pytest.raises(TypeError):
        quantize_rows(q)
    with pytest.raises(ValueError):
        quantize_rows(wi[:, :0])
    with pytest.raises(ValueError):
        int8_linear(x[:, 1:], q, s)
    with pytest.raises(RuntimeError, match="no backward"):
        int8_linear(x.detach().requires_grad_(), q, s)
    with pytest.raises(RuntimeError, match="no backward"):
        int8_linear(x, q, s, bias=torch.zeros(32, dtype=BF16, device="cuda", requires_grad=True))
    with pytest.raises(RuntimeError, match="no backward"):
        int8_matmul(q, s.clone().requires_grad_(), q, s)


def test_calls_from_several_threads():
    import threading

    t = ff_inputs(300, 64, 200, 48, BF16, True)
    args = [t[n] for n in ("x", "w_in", "w_out", "b_in", "b_out")]
    layer = Int8Linear.from_weight(t["w_in"])
    want = gated_feed_forward(*args), layer(t["x"]), dropout(t["x"], 0.3, 1)
    torch.cuda.synchronize()
    wrong = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = gated_feed_forward(*args), layer(t["x"]), dropout(t["x"], 0.3, 1)
                s.synchronize()
                wrong.extend(i for i in range(3) if not torch.equal(got[i], want[i]))

    threads = [threading.Thread(target=work) for _ in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


FIRST_CALL_CAPTURED = """
import torch
from guass_b200.dropout import dropout
from guass_b200.feedforward import gated_feed_forward
from guass_b200.int8 import Int8Linear, int8_linear
x = torch.randn(40, 64, device="cuda").bfloat16().requires_grad_()
w = torch.randn(256, 64, device="cuda").bfloat16() * 0.1
v = torch.randn(64, 128, device="cuda").bfloat16() * 0.1
dy = torch.randn(40, 64, device="cuda").bfloat16()
q = torch.randint(-127, 128, (48, 64), dtype=torch.int8, device="cuda")
s = torch.rand(48, device="cuda")

def step():
    y = dropout(gated_feed_forward(x, w, v, dropout_p=0.1, seed=3), 0.2, 4, residual=x)
    g, = torch.autograd.grad(y, [x], dy)
    return y.detach(), g, int8_linear(x.detach(), q, s)

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, step()))
print("ok")
"""


def test_first_call_of_a_process_may_be_captured():
    import subprocess
    import sys
    from pathlib import Path

    r = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], capture_output=True, text=True, timeout=300,
                       cwd=Path(__file__).resolve().parent.parent)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stderr[-2000:]
