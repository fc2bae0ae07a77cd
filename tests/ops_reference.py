"""The operators of trainable heads in 64 bits on the CPU, with bounds on how far a
correct evaluation may be off, element by element.

The bounds follow the errors through the formulas: u is half a unit in the last place of
the type (each rounding to it), a sum of k products formed in fp32 is off by at most (k + 32)
2^-23 of the sum of their magnitudes (one ulp an addition, so that truncating matrix
cores are inside it, and 32 for the dropped products of the pieces and the joining of slices),
the activation and its derivative by 2^-20 of their scale. |act'| <= 1.13 and |act''| <= 1
for the three activations."""
import math

import torch

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_ULP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
# half the distance of the smallest numbers that the type holds
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -25}
SLOPE, BEND, ACT = 1.13, 1.0, 2.0 ** -20


def act64(kind, g):
    if kind == "tanh":
        a = torch.tanh(g)
        return a, 1 - a * a
    if kind == "silu":
        p = torch.sigmoid(g)
        return g * p, p * (1 + g * (1 - p))
    p = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
    return g * p, p + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def gamma(k):
    return (k + 32) * 2.0 ** -23


def gated(dtype, act, x, wg, wu, wd, dy=None):
    """{name: (value, bound)} of y and, with dy, of dx, dwg, dwu and dwd; float64 inputs
    that the type holds."""
    u, tiny = HALF_ULP[dtype], TINY[dtype]
    n, d = x.shape
    f, o = wd.shape
    ax, ag, au, ad = x.abs(), wg.abs(), wu.abs(), wd.abs()
    g, up = x @ wg, x @ wu
    bg, bu = gamma(d) * (ax @ ag), gamma(d) * (ax @ au)
    a, da = act64(act, g)
    h = a * up
    bh = SLOPE * up.abs() * bg + a.abs() * bu + SLOPE * bg * bu + ACT * (1 + a.abs()) * up.abs()
    bh = bh + u * (h.abs() + bh) + tiny
    y = h @ wd
    by = bh @ ad + gamma(f) * ((h.abs() + bh) @ ad)
    out = {"y": (y, by + u * (y.abs() + by) + tiny)}
    if dy is None:
        return out
    ady = dy.abs()
    dh = dy @ wd.T
    bdh = gamma(o) * (ady @ ad.T)
    du, dg = dh * a, dh * up * da
    ba, bda = SLOPE * bg + ACT * (1 + a.abs()), BEND * bg + ACT * (1 + g.abs())
    bdu = a.abs() * bdh + ba * (dh.abs() + bdh)
    bdg = (up * da).abs() * bdh + (da.abs() * bu + up.abs() * bda + bu * bda) * (dh.abs() + bdh)
    bdu = bdu + u * (du.abs() + bdu) + tiny
    bdg = bdg + u * (dg.abs() + bdg) + tiny
    pdu, pdg = du.abs() + bdu, dg.abs() + bdg
    for name, v, b in (
            ("dx", dg @ wg.T + du @ wu.T, bdg @ ag.T + bdu @ au.T + gamma(2 * f) * (pdg @ ag.T + pdu @ au.T)),
            ("dwg", x.T @ dg, ax.T @ bdg + gamma(n) * (ax.T @ pdg)),
            ("dwu", x.T @ du, ax.T @ bdu + gamma(n) * (ax.T @ pdu)),
            ("dwd", h.T @ dy, bh.T @ ady + gamma(n) * ((h.abs() + bh).T @ ady))):
        out[name] = (v, b + u * (v.abs() + b) + tiny)
    return out


def embed(dtype, ids, table, scale):
    """(value, bound) of the lookup."""
    ok = (ids >= 0) & (ids < len(table))
    v = torch.where(ok[:, None], table[torch.where(ok, ids, 0).long()] * scale, 0.0)
    return v, (HALF_ULP[dtype] + 2.0 ** -24) * v.abs() + TINY[dtype]


def embed_grad(dtype, ids, dout, vocab, scale):
    """(value, bound) of the table's gradient: a sum of k rows, then the scale, then the type."""
    ok = (ids >= 0) & (ids < vocab)
    rows, at = dout[ok], ids[ok].long()
    v = torch.zeros(vocab, dout.shape[1], dtype=torch.float64).index_add_(0, at, rows)
    mag = torch.zeros_like(v).index_add_(0, at, rows.abs())
    k = torch.bincount(at, minlength=vocab)[:, None]
    b = (k + 2) * 2.0 ** -24 * mag * abs(scale)
    v = v * scale
    return v, b + HALF_ULP[dtype] * (v.abs() + b) + TINY[dtype]
