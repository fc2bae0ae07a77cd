"""Group norm, 8-bit checkpoints and products in 8-bit integers in 64 bits on the CPU, with bounds on how
far a correct evaluation may be off, element by element.

What is held in 8 bits has no bound: integers, units and scales follow from their definitions bit by bit.
The others: a sum that is formed in fp32, each value passing at most k additions, is off by at most (k + 32) 2^-23
of the sum of magnitudes; a product, difference or quotient rounds by 2^-24 of itself; activations as in
ops_reference.py."""
import math

import torch

import ops_reference as ref

E32 = 2.0 ** -24


def act64(kind, g):
    return (g, torch.ones_like(g)) if kind == "none" else ref.act64(kind, g)


def act_bound(kind, v, db, slope):
    """Of act(g) (v, slope SLOPE) or act'(g) (v = g, slope BEND) from the bound db of g."""
    if kind == "none":
        return db if slope == ref.SLOPE else torch.zeros_like(db)
    return slope * db + ref.ACT * (1 + v.abs())


# ---- checkpoints ------------------------------------------------------------------------------
def fields(x):
    """(q, field of each group) of x, float64 of numbers that fp32 holds: [rows][wide], [rows][wide / 32]."""
    n, cols = x.shape
    wide = -(-cols // 32) * 32
    g = torch.zeros(n, wide, dtype=torch.float64)
    g[:, :cols] = x
    g = g.reshape(n, wide // 32, 32)
    top = g.abs().amax(2)
    power = torch.full_like(top, -127.0)  # floor(log2 top), at least -127
    for k in range(-126, 128):
        power = torch.where(top >= 2.0 ** k, float(k), power)
    good = torch.isfinite(top)
    unit = torch.pow(torch.tensor(2.0, dtype=torch.float64), power - 6)[..., None]
    q = torch.where(good[..., None], torch.round(g / unit).clamp(-127, 127), 0.0)
    field = torch.where(good, power + 127, 255.0).to(torch.uint8)
    return q.reshape(n, wide).to(torch.int8), field


def restored(x):
    q, field = fields(x)
    unit = torch.pow(torch.tensor(2.0, dtype=torch.float64), field.double() - 133)
    unit = torch.where(field == 255, math.nan, unit).repeat_interleave(32, 1)
    return (q.double() * unit)[:, :x.shape[1]]


# ---- products ----------------------------------------------------------------------------------
def rows8(x):
    """(q, scale) of the rows of x, float64 of numbers that fp32 holds: the scales are fp32 numbers."""
    top = x.abs().amax(1, keepdim=True)
    bad = ~torch.isfinite(top)
    some = (top >= 2.0 ** -119) & ~bad
    safe = torch.where(some, top, 1.0)
    # (a quotient of two fp32 numbers, rounded to 53 bits and then to 24, is rounded as at once)
    inv = (127.0 / safe).float().double()
    scale = torch.where(some, (safe / 127.0).float().double(), 0.0)
    q = torch.where(some, torch.round(torch.where(some, x, 0.0) * inv), 0.0)
    return q, torch.where(bad, math.nan, scale)


def linear8(dtype, act, x, w, w_scale, up=None, up_scale=None):
    """(value, bound): w, up the integers [d_out][d_in] and their scales."""
    q, scale = rows8(x)

    def side(m, s):
        g = (q @ m.double().T) * scale * s.double()
        return g, 4 * E32 * g.abs() + 2.0 ** -148

    g, bg = side(w, w_scale)
    v = act64(act, g)[0]
    b = act_bound(act, v, bg, ref.SLOPE)
    if up is not None:
        u, bu = side(up, up_scale)
        b = v.abs() * bu + (u.abs() + bu) * b + 2 * E32 * (v * u).abs()
        v = v * u
    return v, b + ref.HALF_ULP[dtype] * (v.abs() + b) + ref.TINY[dtype]


# ---- group norm ---------------------------------------------------------------------------------
def norm(dtype, act, x, gamma, beta, frames, groups, eps, dy=None, at=None):
    """{name: (value, bound)} of y, stats and, with dy, dx, dgamma, dbeta; frames: (first, count) of each; at: what
    the gradients are taken at in place of x. Rows of no frame are NaN in y and dx."""
    n, ch = x.shape
    per = ch // groups
    u, tiny = ref.HALF_ULP[dtype], ref.TINY[dtype]
    gm, bt = gamma.reshape(groups, per), beta.reshape(groups, per)
    first, each = frames[0]
    if each and all(f == (first + k * each, each) for k, f in enumerate(frames)):
        batches = [(0, len(frames), first, each)]  # (all at once)
    else:
        batches = [(f, 1, first, count) for f, (first, count) in enumerate(frames)]
    out = {"y": [torch.full_like(x, math.nan) for _ in range(2)],
           "stats": [x.new_zeros(len(frames), groups, 2) for _ in range(2)]}
    if dy is not None:
        out["dx"] = [torch.full_like(x, math.nan) for _ in range(2)]
        for k in ("dgamma", "dbeta"):
            out[k] = [x.new_zeros(groups, per) for _ in range(2)]
    sums = (n + 32) * 2.0 ** -23
    for f, many, first, count in batches:
        if not count:
            continue
        rows, shape = slice(first, first + many * count), (many, count, groups, per)
        a = x[rows].reshape(shape)
        number = count * per
        # a value passes at most 32 additions in its thread's batch, a join for every fourth row,
        # and 256 parts of a block
        g = (min(number, 300 + count // 4) + 32) * 2.0 ** -23

        def mean(v):
            return v.mean((1, 3), keepdim=True)

        m = mean(a)
        bm = g * mean(a.abs())
        var = mean((a - m) ** 2)
        bvar = g * var + 2 * bm * var.sqrt() + bm ** 2
        r = (var + eps) ** -0.5
        br = ((var - bvar).clamp(min=0) + eps) ** -0.5 - r + 4 * E32 * r
        out["stats"][0][f:f + many] = torch.stack([m, r], -1).reshape(many, groups, 2)
        out["stats"][1][f:f + many] = torch.stack([bm + E32 * m.abs(), br], -1).reshape(many, groups, 2)

        def value(t):
            d = t - m
            v = d * r
            bv = (E32 * d.abs() + bm) * (r + br) + d.abs() * br + 2 * E32 * v.abs()
            z = gm * v + bt
            return v, bv, z, gm.abs() * bv + 3 * E32 * ((gm * v).abs() + bt.abs())

        v, bv, z, bz = value(a)
        y = act64(act, z)[0]
        by = act_bound(act, y, bz, ref.SLOPE)
        out["y"][0][rows] = y.reshape(many * count, ch)
        out["y"][1][rows] = (by + u * (y.abs() + by) + tiny).reshape(many * count, ch)
        if dy is None:
            continue
        if at is not None:
            v, bv, z, bz = value(at[rows].reshape(shape))
        d = dy[rows].reshape(shape)
        da = act64(act, z)[1]
        dz = d * da
        bdz = d.abs() * act_bound(act, z, bz, ref.BEND) + 2 * E32 * dz.abs()
        w, bw = gm * dz, gm.abs() * bdz + 2 * E32 * (gm * dz).abs()
        wv, bwv = w * v, bw * (v.abs() + bv) + w.abs() * bv + 2 * E32 * (w * v).abs()
        s1, b1 = mean(w), mean(bw) + g * mean(w.abs() + bw)
        s2, b2 = mean(wv), mean(bwv) + g * mean(wv.abs() + bwv)
        inner = w - s1 - v * s2
        bi = bw + b1 + v.abs() * b2 + bv * (s2.abs() + b2) + 4 * E32 * (w.abs() + s1.abs() + (v * s2).abs())
        dx = r * inner
        bx = (r + br) * bi + br * inner.abs() + 2 * E32 * dx.abs()
        out["dx"][0][rows] = dx.reshape(many * count, ch)
        out["dx"][1][rows] = (bx + u * (dx.abs() + bx) + tiny).reshape(many * count, ch)
        dv, bdv = dz * v, bdz * (v.abs() + bv) + dz.abs() * bv + 2 * E32 * (dz * v).abs()
        for k, t, b in (("dgamma", dv, bdv), ("dbeta", dz, bdz)):
            out[k][0] += t.sum((0, 1))
            out[k][1] += (b + sums * (t.abs() + b)).sum((0, 1))
    if dy is not None:
        for k in ("dgamma", "dbeta"):
            t, b = (z.reshape(ch) for z in out[k])
            out[k] = [t, b + u * (t.abs() + b) + tiny]
    return {k: tuple(v) for k, v in out.items()}
