"""64-bit definitions of the block operators and the error their kernels may
have, for the tests.

Roundings: storing a value as type t moves it by at most half a step,
``eps(t) / 2`` relative (or half the smallest subnormal); an fp32 sum of n
products on the tensor cores by at most n * 2**-23 of the sum of the
magnitudes (one truncation per addition); an activation evaluated in fp32 by
at most 2**-19 of its argument, which is a thousandth of the fp16 step it is
rounded to.  The bounds below carry these through the formulas to first order;
SLACK covers the products of two errors.
"""
from __future__ import annotations

import numpy as np
import torch

SLACK = 1.02
ACT_ERR = 2.0 ** -19
SUM_ERR = 2.0 ** -23


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(v, dtype):
    """Largest move of the values ``v`` when stored as ``dtype``."""
    sub = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return (v.abs() * half_step(dtype)).clamp_min(sub)


def philox(counter, key):
    """Philox-4x32-10 on python integers: counter (4 words), key (2 words)."""
    c, k = list(counter), list(key)
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def keep_mask(rows, cols, p, seed, site):
    """[rows, cols] bool on the CPU: which elements the dropout rule keeps."""
    m32 = np.uint64(0xFFFFFFFF)
    blocks = -(-cols // 4)
    r, b = np.meshgrid(np.arange(rows, dtype=np.uint64), np.arange(blocks, dtype=np.uint64), indexing="ij")
    c = [b, r & m32, np.full_like(b, site), r >> np.uint64(32)]
    k0, k1 = np.uint64(seed & 0xFFFFFFFF), np.uint64(seed >> 32 & 0xFFFFFFFF)
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ k0, p1 & m32, (p0 >> np.uint64(32)) ^ c[3] ^ k1, p0 & m32]
        k0, k1 = (k0 + np.uint64(0x9E3779B9)) & m32, (k1 + np.uint64(0xBB67AE85)) & m32
    words = np.stack(c, -1).reshape(rows, 4 * blocks)[:, :cols]
    return torch.from_numpy(words >= np.uint64(min(round(p * 2 ** 32), 2 ** 32 - 1)))


def activation(name, g):
    """(value, slope, largest |curvature|) in the type of ``g``."""
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-g * 0.5 ** 0.5)
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (2 * np.pi) ** -0.5, 0.8
    sig = torch.sigmoid(g)
    return g * sig, sig * (1 + g * (1 - sig)), 0.5


def feed_forward(x, w_in, w_out, b_in, b_out, act, keep, dy, dtype):
    """Exact outputs and bounds: {name: (value, bound)}.  ``keep``: the hidden
    mask times 1 / (1 - p), or None."""
    x, w_in, w_out, b_in, b_out, dy = (None if t is None else t.detach().double().cpu()
                                       for t in (x, w_in, w_out, b_in, b_out, dy))
    m, d = x.shape
    o, f = w_out.shape
    keep = torch.ones(m, f, dtype=torch.float64) if keep is None else keep.double()
    u = x @ w_in.t() + (0 if b_in is None else b_in)
    eu = (d + 1) * SUM_ERR * (x.abs() @ w_in.abs().t() + (0 if b_in is None else b_in.abs()))
    v, g = u[:, :f], u[:, f:]
    ev, eg = eu[:, :f], eu[:, f:]
    a, slope, curve = activation(act, g)
    h = v * a * keep
    eh = keep * (a.abs() * ev + v.abs() * (1.13 * eg + ACT_ERR * g.abs())) + h.abs() * 2.0 ** -21
    eh = eh + rounding(h, dtype)
    y = h @ w_out.t() + (0 if b_out is None else b_out)
    ey = eh @ w_out.abs().t() + (f + 1) * SUM_ERR * (h.abs() @ w_out.abs().t() + (0 if b_out is None else b_out.abs()))
    out = dict(y=(y, SLACK * (ey + rounding(y, dtype))))
    if dy is None:
        return out
    dh = dy @ w_out * keep
    edh = keep * (o * SUM_ERR * (dy.abs() @ w_out.abs())) + dh.abs() * 2.0 ** -22
    dv, dg = dh * a, dh * v * slope
    edv = a.abs() * edh + dh.abs() * (1.13 * eg + ACT_ERR * (1 + g.abs()))
    edg = (v * slope).abs() * edh + (dh * slope).abs() * ev + (dh * v).abs() * (curve * eg + ACT_ERR * (1 + g.abs()))
    du, edu = torch.cat([dv, dg], 1), torch.cat([edv, edg], 1)
    edu = edu + du.abs() * 2.0 ** -21 + rounding(du, dtype)

    def result(value, error):
        return value, SLACK * (error + rounding(value, dtype))

    out["dx"] = result(du @ w_in, edu @ w_in.abs() + 2 * f * SUM_ERR * (du.abs() @ w_in.abs()))
    out["dw_in"] = result(du.t() @ x, edu.t() @ x.abs() + m * SUM_ERR * (du.abs().t() @ x.abs()))
    out["dw_out"] = result(dy.t() @ h, dy.abs().t() @ eh + m * SUM_ERR * (dy.abs().t() @ h.abs()))
    out["db_in"] = result(du.sum(0), edu.sum(0) + m * SUM_ERR * du.abs().sum(0))
    out["db_out"] = result(dy.sum(0), m * SUM_ERR * dy.abs().sum(0))
    return out


def quantise(x):
    """(q, scale) of the row quantisation's definition, on fp32 steps."""
    x = x.detach().float().cpu()
    top = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    zero = bad | (top < 2.0 ** -100)
    inv = torch.where(zero, torch.zeros_like(top), torch.full_like(top, 127.0) / top)
    q = torch.where(zero[..., None], torch.zeros_like(x), (torch.nan_to_num(x) * inv[..., None]).round())
    scale = torch.where(zero, torch.zeros_like(top), top / 127.0)
    return q.to(torch.int8), torch.where(bad, torch.full_like(top, float("nan")), scale)
