"""Measured cases of the transformer-block operators.

Three operators of the block that carries the Gaussian adapters:

* ``ff``: the gated feed-forward block (``guass_b200.feedforward``), forward
  alone or with the gradients of the input (frozen weights, which is how the
  adapters are trained) or of every input;
* ``dropout``: counter-based dropout whose mask is never stored
  (``guass_b200.dropout``), forward and backward;
* ``int8``: the product in 8-bit integers with a scale for each token and each
  output channel (``guass_b200.int8``), the serving form of a merged weight.

With ``own`` false ``run`` evaluates them in elementary torch operations,
with ``own`` true through the framework.  ``exact`` is the definition in 64
bits.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MASK32 = 0xFFFFFFFF


# ---------------------------------------------------------------------------
# cases

def listed():
    return [
        # one token through the widest block: serving, where latency counts
        dict(name="ff-token", op="ff", tokens=1, dim=1280, hidden=5120, dtype="bf16", act="gelu", bias=True, p=0.0,
             mode="infer"),
        # the 8x8 latent of the middle block at batch 1: few rows, a wide block, fp16 serving
        dict(name="ff-64", op="ff", tokens=64, dim=1280, hidden=5120, dtype="fp16", act="gelu", bias=True, p=0.0,
             mode="infer"),
        # 64x64 latents at batch 4, the narrowest and longest block of an adapter training step (frozen weights)
        dict(name="ff-adapter-16384", op="ff", tokens=16384, dim=320, hidden=1280, dtype="bf16", act="gelu", bias=True,
             p=0.0, mode="adapter"),
        # 32x32 latents at batch 4, adapter training with dropout on the hidden activations
        dict(name="ff-adapter-4096", op="ff", tokens=4096, dim=640, hidden=2560, dtype="bf16", act="gelu", bias=True,
             p=0.1, mode="adapter"),
        # 16x16 latents at batch 4, the block trained whole, SiLU gate and no biases (the language-model form)
        dict(name="ff-full-1024", op="ff", tokens=1024, dim=1280, hidden=5120, dtype="fp16", act="silu", bias=False,
             p=0.0, mode="full"),
        # odd sizes throughout (no row of any operand on a 16-byte boundary), every gradient
        dict(name="ff-full-odd", op="ff", tokens=1003, dim=333, hidden=1001, dtype="bf16", act="gelu", bias=True,
             p=0.2, mode="full"),
        # the text embedding of one prompt
        dict(name="dropout-text", op="dropout", rows=77, cols=768, dtype="bf16", p=0.1, residual=False, strided=False),
        # a residual branch of the 64x64 blocks at batch 16
        dict(name="dropout-residual", op="dropout", rows=65536, cols=640, dtype="bf16", p=0.1, residual=True,
             strided=False),
        # odd sizes, a transposed input, fp32
        dict(name="dropout-odd", op="dropout", rows=4099, cols=333, dtype="fp32", p=0.5, residual=False, strided=True),
        # the time embedding's projections: one row for each sample of a batch of 4
        dict(name="int8-rows-4", op="int8", rows=4, k=1280, n=1280, dtype="bf16", bias=True),
        # odd sizes: three prompts of 77 tokens, fp32 in and out
        dict(name="int8-odd", op="int8", rows=231, k=333, n=1001, dtype="fp32", bias=True),
        # the widest feed-forward projection at 16384 tokens
        dict(name="int8-16384", op="int8", rows=16384, k=1280, n=10240, dtype="bf16", bias=True),
    ]


def _between(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["ff", "ff", "dropout", "int8"])
    if op == "ff":
        if rng.random() < 0.6:
            dim = rng.choice([320, 640, 1280])
            hidden = 4 * dim
        else:
            dim, hidden = _between(rng, 16, 1280), _between(rng, 16, 5120)
        mode = rng.choice(["infer", "adapter", "full"])
        most = int(1.2e11 / ({"infer": 6, "adapter": 12, "full": 18}[mode] * dim * hidden))
        return dict(op=op, tokens=_between(rng, 1, min(16384, most)), dim=dim, hidden=hidden,
                    dtype=rng.choice(["bf16", "fp16"]), act=rng.choice(["gelu", "silu"]), bias=rng.random() < 0.7,
                    p=rng.choice([0.0, 0.1, 0.3]), mode=mode)
    if op == "dropout":
        cols = _between(rng, 1, 10240)
        return dict(op=op, rows=_between(rng, 1, min(65536, 41_000_000 // max(cols, 4))), cols=cols,
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), p=rng.choice([0.05, 0.1, 0.5, 0.9]),
                    residual=rng.random() < 0.5, strided=rng.random() < 0.3)
    k, n = _between(rng, 16, 5120), _between(rng, 16, 10240)
    most = min(16384, int(2.1e11 / (k * n)), 160_000_000 // n, 80_000_000 // k)
    return dict(op=op, rows=_between(rng, 1, most), k=k, n=n, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                bias=rng.random() < 0.7)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "ff":
        m, d, f = case["tokens"], case["dim"], case["hidden"]
        weights = 3 * d * f + (2 * f + d if case["bias"] else 0)
        # forward: x, the weights, y; then dy and dx; then the weights' gradients
        n = 2 * m * d + weights
        n += {"infer": 0, "adapter": 2 * m * d, "full": 2 * m * d + weights}[case["mode"]]
        return {"bytes": size * n, "flops": {"infer": 6, "adapter": 12, "full": 18}[case["mode"]] * m * d * f}
    if case["op"] == "dropout":
        # x, y and dy, dx, and the residual; ten rounds of the generator for every four elements, in each direction
        n = case["rows"] * case["cols"]
        return {"bytes": size * n * (5 if case["residual"] else 4), "flops": 2 * n}
    m, k, n = case["rows"], case["k"], case["n"]
    return {"bytes": size * (m * k + m * n + (n if case["bias"] else 0)) + n * k + 4 * n, "flops": 2 * m * n * k}


# ---------------------------------------------------------------------------
# inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    s = dict(case=case, op=case["op"])
    if case["op"] == "ff":
        m, d, f = case["tokens"], case["dim"], case["hidden"]
        # x is the output of a layer norm; dy is the gradient of a scaled loss
        s.update(x=normal(m, d), w_in=normal(2 * f, d, std=d ** -0.5), w_out=normal(d, f, std=f ** -0.5),
                 b_in=normal(2 * f, std=0.1) if case["bias"] else None,
                 b_out=normal(d, std=0.1) if case["bias"] else None)
        if case["mode"] != "infer":
            s["dy"] = normal(m, d)
            s["x"].requires_grad_()
        if case["mode"] == "full":
            for name in ("w_in", "w_out", "b_in", "b_out"):
                if s[name] is not None:
                    s[name].requires_grad_()
        # a training step's seed lives on the device, where a captured step can advance it
        s["seed"] = torch.tensor([seed * 2654435761 % (1 << 62)], dtype=torch.int64, device="cuda")
        s["site"] = 3
    elif case["op"] == "dropout":
        shape = (case["rows"], case["cols"])
        s["x"] = (normal(*shape[::-1]).t() if case["strided"] else normal(*shape)).requires_grad_()
        s["residual"] = normal(*shape).requires_grad_() if case["residual"] else None
        s["dy"] = normal(*shape)
        s["seed"], s["site"] = seed * 2654435761 % (1 << 62), 5
    else:
        m, k, n = case["rows"], case["k"], case["n"]
        # activations with a few channels far above the others, as transformers have them
        loud = 1.0 + 9.0 * (torch.rand(k, generator=g, device="cuda") < 0.01).float()
        s["x"] = (torch.randn(m, k, generator=g, device="cuda") * loud).to(dt)
        w = torch.randn(n, k, generator=g, device="cuda") * k ** -0.5
        s["w_scale"] = w.abs().amax(1) / 127.0
        # the 8-bit weight as the framework keeps it: rows that start on 16-byte boundaries
        s["w_q"] = torch.zeros(n, -(-k // 16) * 16, dtype=torch.int8, device="cuda")[:, :k]
        s["w_q"].copy_(torch.round(w / s["w_scale"][:, None]))
        s["bias"] = normal(n, std=0.1) if case["bias"] else None
    return s


# ---------------------------------------------------------------------------
# plain forms

def _random_words(rows, cols, seed, site):
    """Philox-4x32-10 (Salmon et al., SC 2011): [rows, cols] words of 32 bits in int64.  Element (r, c) is word c % 4 of
    counter (c // 4, r, site, r >> 32) under the key (low, high) of the 64-bit seed."""
    dev = "cuda"
    c0 = torch.arange(-(-cols // 4), device=dev).view(1, -1).expand(rows, -1)
    r = torch.arange(rows, device=dev).view(-1, 1)
    c1, c3 = (r & MASK32).expand_as(c0), (r >> 32).expand_as(c0)
    c2 = torch.full_like(c0, site & MASK32)
    k0, k1 = seed & MASK32, (seed >> 32) & MASK32
    for _ in range(10):  # the generator's rounds
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64-bit products: the words wrap as unsigned ones do
        c0, c1, c2, c3 = ((p1 >> 32) & MASK32) ^ c1 ^ k0, p1 & MASK32, ((p0 >> 32) & MASK32) ^ c3 ^ k1, p0 & MASK32
        k0, k1 = (k0 + 0x9E3779B9) & MASK32, (k1 + 0xBB67AE85) & MASK32
    return torch.stack([c0, c1, c2, c3], -1).view(rows, -1)[:, :cols]


def _keep_scale(rows, cols, p, seed, site):
    """1 / (1 - p) where an element is kept, 0 where it is dropped (fp32)."""
    keep = _random_words(rows, cols, seed, site) >= round(p * 2 ** 32)
    return keep.float() * (1.0 / (1.0 - p))


def _plain_ff(s):
    c = s["case"]
    x, w_in, w_out = (s[n].detach().float() for n in ("x", "w_in", "w_out"))
    dt, f = s["x"].dtype, c["hidden"]
    u = x @ w_in.t()
    if c["bias"]:
        u = u + s["b_in"].detach().float()
    a, g = u[:, :f], u[:, f:]
    if c["act"] == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * 0.5 ** 0.5))
        act, slope = g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (2.0 * math.pi) ** -0.5
    else:
        sig = 1.0 / (1.0 + torch.exp(-g))
        act, slope = g * sig, sig * (1.0 + g * (1.0 - sig))
    keep = _keep_scale(c["tokens"], f, c["p"], s["seed"], s["site"]) if c["p"] > 0 else 1.0
    h = a * act * keep
    y = h @ w_out.t()
    if c["bias"]:
        y = y + s["b_out"].detach().float()
    if c["mode"] == "infer":
        return y.to(dt)
    dy = s["dy"].float()
    dh = dy @ w_out * keep
    du = torch.cat([dh * act, dh * a * slope], 1)
    out = dict(y=y.to(dt), dx=(du @ w_in).to(dt))
    if c["mode"] == "full":
        out.update(dw_in=(du.t() @ x).to(dt), dw_out=(dy.t() @ h).to(dt))
        if c["bias"]:
            out.update(db_in=du.sum(0).to(dt), db_out=dy.sum(0).to(dt))
    return out


def _plain_dropout(s):
    c = s["case"]
    keep = _keep_scale(c["rows"], c["cols"], c["p"], s["seed"], s["site"])
    dt, x, dy = s["x"].dtype, s["x"].detach().float(), s["dy"]
    y = x * keep
    if c["residual"]:
        y = y + s["residual"].detach().float()
    out = dict(y=y.to(dt), dx=(dy.float() * keep).to(dt))
    if c["residual"]:
        out["dresidual"] = dy.clone()
    return out


def _plain_int8(s):
    x = s["x"].float()
    most = x.abs().amax(1, keepdim=True)
    scale = most / 127.0
    q = torch.round(x * torch.where(most > 0, 127.0 / most, 0.0))
    y = (q.double() @ s["w_q"].t().double()).float() * scale * s["w_scale"]  # whole numbers past 24 bits: 64-bit sums
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


# ---------------------------------------------------------------------------
# one pass

def _own_ff(s):
    from guass_b200.feedforward import gated_feed_forward

    c = s["case"]
    leaves = ["x"] if c["mode"] == "adapter" else ["x", "w_in", "w_out"] + (["b_in", "b_out"] if c["bias"] else [])
    y = gated_feed_forward(s["x"], s["w_in"], s["w_out"], s["b_in"], s["b_out"], activation=c["act"],
                           dropout_p=c["p"], seed=s["seed"], site=s["site"])
    if c["mode"] == "infer":
        return y
    grads = torch.autograd.grad(y, [s[n] for n in leaves], s["dy"])
    return dict(y=y, **{"d" + n: g for n, g in zip(leaves, grads)})


def _own_dropout(s):
    from guass_b200.dropout import dropout

    leaves = ["x"] + (["residual"] if s["residual"] is not None else [])
    y = dropout(s["x"], s["case"]["p"], s["seed"], site=s["site"], residual=s["residual"])
    return dict(y=y, **{"d" + n: g for n, g in zip(leaves, torch.autograd.grad(y, [s[n] for n in leaves], s["dy"]))})


def _own_int8(s):
    from guass_b200.int8 import int8_linear

    return int8_linear(s["x"], s["w_q"], s["w_scale"], s["bias"])


def run(state):
    if own:
        return {"ff": _own_ff, "dropout": _own_dropout, "int8": _own_int8}[state["op"]](state)
    with torch.no_grad():
        return {"ff": _plain_ff, "dropout": _plain_dropout, "int8": _plain_int8}[state["op"]](state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits

def _words_by_halves(rows, cols, seed, site):
    """The same generator on 16-bit halves, so that no product passes 63 bits."""
    def product(a, b):  # (high, low) 32 bits of a * b
        al, ah, bl, bh = a & 0xFFFF, a >> 16, b & 0xFFFF, b >> 16
        mid = ah * bl + ((al * bl) >> 16)
        low_mid = al * bh + (mid & 0xFFFF)
        return ah * bh + (mid >> 16) + (low_mid >> 16), ((low_mid & 0xFFFF) << 16) | ((al * bl) & 0xFFFF)

    blocks = (cols + 3) // 4
    i = torch.arange(rows * blocks, device="cuda")
    row = i // blocks
    x = [i - row * blocks, row & MASK32, torch.zeros_like(i) + (site & MASK32), row >> 32]
    for n in range(10):
        ka = ((seed & MASK32) + n * 0x9E3779B9) & MASK32
        kb = ((seed >> 32 & MASK32) + n * 0xBB67AE85) & MASK32
        h0, l0 = product(x[0], 0xD2511F53)
        h1, l1 = product(x[2], 0xCD9E8D57)
        x = [h1 ^ x[1] ^ ka, l1, h0 ^ x[3] ^ kb, l0]
    return torch.stack(x, 1).reshape(rows, 4 * blocks)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)

    def wide(name):
        t = s[name]
        return None if t is None else t.detach().double()

    if case["op"] == "int8":
        # the quantised activations are the operator's own whole numbers: scales and rounding are defined in fp32
        x = s["x"].to(torch.float32)
        top = x.abs().max(1).values
        inv = torch.zeros_like(top)
        inv[top > 0] = torch.full_like(top[top > 0], 127.0) / top[top > 0]
        q = (x * inv[:, None]).round().double()
        y = torch.einsum("mk,nk->mn", q, wide("w_q")) * (top / 127.0).double()[:, None] * wide("w_scale")[None]
        return y if s["bias"] is None else y + wide("bias")

    if case["op"] == "dropout":
        kept = _words_by_halves(case["rows"], case["cols"], s["seed"], s["site"]) >= round(case["p"] * 2 ** 32)
        y = torch.where(kept, wide("x") / (1.0 - case["p"]), 0.0)
        out = dict(y=y, dx=torch.where(kept, wide("dy") / (1.0 - case["p"]), 0.0))
        if case["residual"]:
            out.update(y=y + wide("residual"), dresidual=wide("dy"))
        return out

    names = ["x"] + (["w_in", "w_out", "b_in", "b_out"] if case["mode"] == "full" else [])
    t = {n: wide(n) for n in ("x", "w_in", "w_out", "b_in", "b_out")}
    names = [n for n in names if t[n] is not None and case["mode"] != "infer"]
    for n in names:
        t[n].requires_grad_()
    value, gate = torch.nn.functional.linear(t["x"], t["w_in"], t["b_in"]).chunk(2, dim=-1)
    h = value * (torch.nn.functional.gelu(gate) if case["act"] == "gelu" else torch.nn.functional.silu(gate))
    if case["p"] > 0:
        kept = _words_by_halves(case["tokens"], case["hidden"], int(s["seed"]), s["site"]) >= round(case["p"] * 2 ** 32)
        h = torch.where(kept, h / (1.0 - case["p"]), 0.0)
    y = torch.nn.functional.linear(h, t["w_out"], t["b_out"])
    if case["mode"] == "infer":
        return y
    grads = torch.autograd.grad(y, [t[n] for n in names], wide("dy"))
    return dict(y=y.detach(), **{"d" + n: g for n, g in zip(names, grads)})
