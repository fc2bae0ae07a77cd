"""Checkpoints in 8 bits, the gated block's gradients from them, 8-bit weights and the products in 8-bit
integers on the GPU: what is held in 8 bits against its definition bit by bit, the rest against 64 bits within the
bounds of ops8_reference.py."""
import math

import pytest
import torch

import ops8_reference as ref8
import ops_reference as ref
from test_gpu_ops import Mat, check, rand, stream

pytestmark = pytest.mark.gpu
TYPES = ["f32", "bf16", "f16"]


@pytest.fixture(scope="module")
def ops(dp):
    return dp.ops.Operators()


def kept_of(dp, rows, cols, tail=64):
    """A checkpoint's buffer with a marker behind it."""
    return torch.full((dp.ops.keep8_bytes(rows, cols) + tail,), 0xA5, dtype=torch.uint8, device="cuda")


def special(gen, dtype, rows, cols):
    """Rows of very different sizes, ties, zeros, subnormal numbers, infinities and NaN."""
    t = ref.TORCH[dtype]
    size = torch.pow(2.0, torch.randint(-20, 15, (rows, 1), generator=gen).double())
    x = torch.randn(rows, cols, generator=gen, dtype=torch.float64) * size
    x[::3] = torch.round(x[::3] / size[::3] * 8) / 16 * size[::3]  # ties
    x[1::7] = 0
    if dtype != "f16":
        x[2::7] *= 2.0 ** -125
        x[3::7] *= 2.0 ** 100
    top = float(torch.finfo(t).max)
    x = x.clamp(-top, top)
    x[4::9, cols // 2] = top
    x[5::9, cols - 1] = math.inf
    x[6::9, 0] = math.nan
    return x.to(t)


# ---- checkpoints ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,pad,skip", [
    (1, 1, 0, 0), (1, 32, 0, 0), (3, 31, 0, 0), (5, 33, 1, 1), (64, 64, 8, 8), (70, 70, 0, 3), (129, 1600, 0, 0),
    (33, 2048, 16, 0), (2, 8193, 5, 0), (1000, 8, 0, 0), (4097, 40, 0, 0)])
def test_checkpoint(ops, dp, dtype, rows, cols, pad, skip):
    gen = torch.Generator().manual_seed(rows + cols)
    host = special(gen, dtype, rows, cols)
    x, kept = Mat(host, pad=pad, skip=skip), kept_of(dp, rows, cols)
    out = Mat(shape=(rows, cols), dtype=dtype, pad=pad, skip=skip, fill=7.0)
    ops.keep8(x.ptr, kept.data_ptr(), rows, cols, dtype, ld_x=x.ld, stream=stream())
    ops.restore8(kept.data_ptr(), out.ptr, rows, cols, dtype, ld_x=out.ld, stream=stream())
    torch.cuda.synchronize()
    q, field = ref8.fields(host.double())
    wide = q.shape[1]
    assert torch.equal(kept[:rows * wide].cpu().view(torch.int8).reshape(rows, wide), q)
    assert torch.equal(kept[rows * wide:-64].cpu().reshape(rows, wide // 32), field)
    assert bool((kept[-64:] == 0xA5).all())
    want = ref8.restored(host.double()).to(ref.TORCH[dtype])
    assert torch.equal(torch.nan_to_num(out.view.cpu().float(), nan=12345.0),
                       torch.nan_to_num(want.float(), nan=12345.0))
    assert out.untouched(7.0)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_restored_in_another_type(ops, dp, dtype):
    """A checkpoint knows no type: what a type can not hold is rounded once."""
    gen = torch.Generator().manual_seed(1)
    host = (torch.randn(50, 100, generator=gen, dtype=torch.float64) * 2.0 ** -14).bfloat16()
    x, kept, out = host.cuda(), kept_of(dp, 50, 100), torch.empty(50, 100, dtype=ref.TORCH[dtype], device="cuda")
    ops.keep8(x.data_ptr(), kept.data_ptr(), 50, 100, "bf16", stream=stream())
    ops.restore8(kept.data_ptr(), out.data_ptr(), 50, 100, dtype, stream=stream())
    assert torch.equal(out.cpu(), ref8.restored(host.double()).to(out.dtype))


def test_checkpoint_past_32_bits(ops, dp):
    """More than 2^32 values: the last rows, whose places pass 32 bits, and the first."""
    rows, cols = 2 ** 21 + 5, 2080
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator().manual_seed(9)
    ends = torch.randn(16, cols, generator=gen).bfloat16()
    x.fill_(1.0)
    x[:8], x[-8:] = ends[:8].cuda(), ends[8:].cuda()
    kept = torch.empty(dp.ops.keep8_bytes(rows, cols), dtype=torch.uint8, device="cuda")
    ops.keep8(x.data_ptr(), kept.data_ptr(), rows, cols, "bf16", stream=stream())
    x.zero_()
    ops.restore8(kept.data_ptr(), x.data_ptr(), rows, cols, "bf16", stream=stream())
    want = ref8.restored(ends.double()).bfloat16()
    assert torch.equal(x[:8].cpu(), want[:8]) and torch.equal(x[-8:].cpu(), want[8:])
    assert bool((x[8:-8] == 1.0).all())


# ---- the gated block from a checkpoint --------------------------------------------------------
def backward8_case(ops, dp, dtype, act, n, d, f, o, pad=0, skip=0, which=("dx", "dwg", "dwu", "dwd")):
    gen = torch.Generator().manual_seed(n + d + f)
    host = {"x": rand(gen, dtype, n, d), "wg": rand(gen, dtype, d, f, d ** -0.5),
            "wu": rand(gen, dtype, d, f, d ** -0.5), "wd": rand(gen, dtype, f, o, f ** -0.5),
            "dy": rand(gen, dtype, n, o)}
    m = {k: Mat(v, pad=pad, skip=skip) for k, v in host.items()}
    outs = {"dx": (n, d), "dwg": (d, f), "dwu": (d, f), "dwd": (f, o)}
    for k, s in outs.items():
        m[k] = Mat(shape=s, dtype=dtype, pad=pad, skip=skip, fill=7.0)
    shape = dp.ops.GatedShape(n, d, f, o, dtype=dtype, act=act, ld_x=m["x"].ld, ld_y=m["dy"].ld,
                              ld_hidden=m["wg"].ld, ld_down=m["wd"].ld)
    kept = kept_of(dp, n, d)
    p = {k: v.ptr for k, v in m.items()}
    ops.keep8(p["x"], kept.data_ptr(), n, d, dtype, ld_x=m["x"].ld, stream=stream())
    given = [p[k] if k in which else 0 for k in outs]
    ops.gated_backward8(shape, kept.data_ptr(), p["wg"], p["wu"], p["wd"], p["dy"], *given, stream=stream())
    torch.cuda.synchronize()
    at = "cuda" if n * f * max(d, o) > 2e9 else "cpu"
    back = ref8.restored(host["x"].double())
    want = ref.gated(dtype, act, back.to(at), *(host[k].double().to(at) for k in ("wg", "wu", "wd", "dy")))
    for k in outs:
        if k in which:
            v, b = want[k]
            check(m[k].view, (v.cpu(), b.cpu()), (k, dtype, act, n, d, f, o))
        else:
            assert bool((m[k].view == 7.0).all())
        assert m[k].untouched(7.0), k
    return {k: m[k].view.clone() for k in outs}


SIZES = [(1, 1, 1, 1), (2, 7, 9, 5), (8, 40, 64, 16), (17, 33, 65, 31), (31, 70, 96, 1), (65, 129, 130, 127),
         (128, 64, 128, 64), (257, 100, 60, 4), (300, 260, 520, 264), (1000, 30, 2100, 5)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,f,o", SIZES)
def test_backward_from_a_checkpoint(ops, dp, dtype, n, d, f, o):
    act = ("silu", "tanh", "gelu")[(n + d) % 3]
    first = backward8_case(ops, dp, dtype, act, n, d, f, o)
    again = backward8_case(ops, dp, dtype, act, n, d, f, o)
    assert all(torch.equal(first[k], again[k]) for k in first)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,skip", [(8, 8), (3, 1)])
def test_backward_from_a_checkpoint_strides(ops, dp, dtype, pad, skip):
    backward8_case(ops, dp, dtype, "silu", 33, 40, 72, 24, pad=pad, skip=skip)
    backward8_case(ops, dp, dtype, "gelu", 70, 41, 71, 3, pad=pad, skip=skip)


@pytest.mark.parametrize("o", [2, 24])
@pytest.mark.parametrize("which", [("dx",), ("dwg", "dwu"), ("dwd",), ("dwg", "dwu", "dwd"), ("dx", "dwd")])
def test_backward_from_a_checkpoint_of_some(ops, dp, which, o):
    backward8_case(ops, dp, "bf16", "silu", 100, 40, 72, o, which=which)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,d,f,o", [(2100, 520, 1040, 264), (5000, 64, 272, 1)])
def test_backward_from_a_checkpoint_large(ops, dp, dtype, n, d, f, o):
    backward8_case(ops, dp, dtype, "silu", n, d, f, o)


def test_backward_from_a_checkpoint_differences(ops, dp):
    """Against differences of the forward, at inputs that the checkpoint holds exactly."""
    n, d, f, o, h = 24, 32, 40, 8, 2.0 ** -3
    gen = torch.Generator().manual_seed(5)
    x = (torch.randint(-96, 96, (n, d), generator=gen).float() / 64).contiguous()
    x[:, 0] = 1.5  # (the unit of every group is then 2^-6, before and after a step)
    w = [(torch.randn(*s, generator=gen) * s[0] ** -0.5) for s in ((d, f), (d, f), (f, o))]
    dy = torch.randn(n, o, generator=gen)
    gx, gdy, gw = x.cuda(), dy.cuda(), [t.cuda() for t in w]
    kept, dx = kept_of(dp, n, d), torch.empty(n, d, device="cuda")
    shape = dp.ops.GatedShape(n, d, f, o, act="tanh")
    ops.keep8(gx.data_ptr(), kept.data_ptr(), n, d, stream=stream())
    ops.gated_backward8(shape, kept.data_ptr(), *(t.data_ptr() for t in gw), gdy.data_ptr(), dx.data_ptr(),
                        stream=stream())
    got = dx.cpu().double()

    def loss(x):
        a, b, c = (t.double() for t in w)
        return ((torch.tanh(x @ a) * (x @ b)) @ c * dy.double()).sum(1)

    for k in range(1, d, 5):
        step = torch.zeros(d, dtype=torch.float64)
        step[k] = h
        # fourth order: the error is h^4 / 30 of a fifth derivative, below 1e-2 of these weights' scale
        slope = (8 * (loss(x.double() + step) - loss(x.double() - step))
                 - (loss(x.double() + 2 * step) - loss(x.double() - 2 * step))) / (12 * h)
        assert (got[:, k] - slope).abs().max() < 1e-2 * (1 + slope.abs().max())


# ---- weights and products -----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,o,pad,skip,more", [(1, 1, 0, 0, 0), (16, 64, 0, 0, 0), (70, 96, 0, 0, 16), (129, 65, 3, 1, 0),
                                               (600, 130, 8, 8, 32), (1023, 17, 0, 0, 0)])
def test_weights(ops, dp, dtype, d, o, pad, skip, more):
    gen = torch.Generator().manual_seed(d + o)
    host = special(gen, dtype, o, d).T.contiguous()  # (special rows become output channels)
    w, ld = Mat(host, pad=pad, skip=skip), (d + 15) // 16 * 16 + more
    q = torch.full((o * ld + 64,), 0x55, dtype=torch.int8, device="cuda")
    scale = torch.full((o + 4,), 7.0, device="cuda")
    ops.weights8(w.ptr, q.data_ptr(), scale.data_ptr(), d, o, dtype, ld_w=w.ld, ld_w8=ld, stream=stream())
    torch.cuda.synchronize()
    want, s = ref8.rows8(host.T.double())
    got = q[:o * ld].cpu().reshape(o, ld)
    assert torch.equal(got[:, :d].double(), want)
    assert bool((got[:, d:ld - more] == 0).all()) and bool((got[:, ld - more:] == 0x55).all())
    assert bool((q[o * ld:] == 0x55).all())
    assert torch.equal(torch.nan_to_num(scale[:o].cpu(), nan=-1.0), torch.nan_to_num(s[:, 0].float(), nan=-1.0))
    assert bool((scale[o:] == 7.0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,o", [(70, 33), (640, 100)])
def test_weights_side_by_side(ops, dp, dtype, d, o):
    """Two matrices whose rows alternate in one array, written one after the other, and multiplied from there."""
    gen = torch.Generator().manual_seed(d)
    whole = (d + 15) // 16 * 16
    host = [rand(gen, dtype, d, o) for _ in range(2)]
    q = torch.full((2 * whole * o + 64,), 0x55, dtype=torch.int8, device="cuda")
    scale = torch.empty(2, o, device="cuda")
    dev = [h.cuda() for h in host]
    for k in (1, 0):
        ops.weights8(dev[k].data_ptr(), q[k * whole:].data_ptr(), scale[k].data_ptr(), d, o, dtype, ld_w8=2 * whole,
                     stream=stream())
    x = rand(gen, dtype, 5, d)
    xd, y = x.cuda(), torch.empty(5, o, dtype=x.dtype, device="cuda")
    shape = dp.ops.Linear8Shape(5, d, o, dtype=dtype, act="silu", ld_w=2 * whole)
    ops.linear8(shape, xd.data_ptr(), q.data_ptr(), scale[0].data_ptr(), y.data_ptr(), d_up=q[whole:].data_ptr(),
                d_up_scale=scale[1].data_ptr(), stream=stream())
    torch.cuda.synchronize()
    want = [ref8.rows8(h.T.double()) for h in host]
    got = q[:2 * whole * o].cpu().reshape(o, 2, whole)
    for k in range(2):
        assert torch.equal(got[:, k, :d].double(), want[k][0]) and bool((got[:, k, d:] == 0).all())
    assert bool((q[2 * whole * o:] == 0x55).all())
    check(y.cpu(), ref8.linear8(dtype, "silu", x.double(), got[:, 0, :d], want[0][1][:, 0], got[:, 1, :d],
                                want[1][1][:, 0]), (dtype, d, o))


def weights(gen, o, d, more=0):
    ld = (d + 15) // 16 * 16 + more
    w = torch.randint(-128, 128, (o, ld), generator=gen).to(torch.int8)  # (what lies past d is not looked at)
    return w, (0.5 + torch.rand(o, generator=gen)) * d ** -0.5 / 127


def linear8_case(ops, dp, dtype, act, n, d, o, gate=False, pad=0, skip=0, more=0, host=None, seed=0):
    gen = torch.Generator().manual_seed(n + d + o + seed)
    host = rand(gen, dtype, n, d) if host is None else host
    x, y = Mat(host, pad=pad, skip=skip), Mat(shape=(n, o), dtype=dtype, pad=pad, skip=skip, fill=7.0)
    w, ws = weights(gen, o, d, more)
    u, us = weights(gen, o, d, more) if gate else (None, None)
    g = [None if t is None else t.cuda() for t in (w, ws, u, us)]
    p = [0 if t is None else t.data_ptr() for t in g]
    shape = dp.ops.Linear8Shape(n, d, o, dtype=dtype, act=act, ld_x=x.ld, ld_y=y.ld, ld_w=w.shape[1])
    ops.linear8(shape, x.ptr, p[0], p[1], y.ptr, d_up=p[2], d_up_scale=p[3], stream=stream())
    torch.cuda.synchronize()
    at = "cuda" if n * o * d > 2e9 else "cpu"
    v, b = ref8.linear8(dtype, act, host.double().to(at), w[:, :d].to(at), ws.to(at),
                        None if u is None else u[:, :d].to(at), None if us is None else us.to(at))
    v, b, got = v.cpu(), b.cpu(), y.view.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(v))
    there = ~torch.isnan(v)
    check(got[there], (v[there], b[there]), (dtype, act, n, d, o, gate))
    assert y.untouched(7.0)
    return y.view.clone()


PRODUCTS = [(1, 1, 1), (1, 2048, 800), (2, 70, 96), (3, 16, 16), (7, 1023, 130), (8, 640, 4100), (9, 129, 33),
            (16, 64, 48), (17, 4100, 65), (33, 2048, 500), (64, 128, 128), (65, 257, 129), (100, 33, 7),
            (130, 1600, 240), (257, 96, 260), (1100, 70, 1040), (2100, 1040, 264)]


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,o", PRODUCTS)
def test_products(ops, dp, dtype, n, d, o, gate):
    act = ("silu", "none", "tanh", "gelu")[(n + d + o) % 4]
    first = linear8_case(ops, dp, dtype, act, n, d, o, gate)
    assert torch.equal(first, linear8_case(ops, dp, dtype, act, n, d, o, gate))


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("n", [1, 2, 4, 5, 15, 16, 17, 32, 33, 48, 49, 63, 64, 65])
@pytest.mark.parametrize("d,o", [(40, 9), (520, 130), (2049, 1031), (12300, 20), (12400, 33), (100, 9000)])
def test_few_rows(ops, dp, n, d, o, gate):
    """Up to 64 rows (kernels of their own): fragments of 16 rows, rows quantised in the same kernel or
    before, k that ends inside a step, waves without a step."""
    for k, dtype in enumerate(TYPES):
        linear8_case(ops, dp, dtype, ("silu", "none", "gelu")[k], n, d, o, gate)


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,skip,more", [(8, 8, 16), (3, 1, 0), (1, 0, 48)])
def test_products_strides(ops, dp, dtype, pad, skip, more, gate):
    for n in (3, 40, 300):
        linear8_case(ops, dp, dtype, "silu", n, 72, 136, gate, pad=pad, skip=skip, more=more)
        linear8_case(ops, dp, dtype, "none", n, 71, 77, gate, pad=pad, skip=skip, more=more)


@pytest.mark.parametrize("n", [5, 70])
@pytest.mark.parametrize("dtype", TYPES)
def test_products_of_special_rows(ops, dp, dtype, n):
    """Rows with an infinity or a NaN are NaN and only they; zeros and numbers near the type's ends."""
    gen = torch.Generator().manual_seed(7)
    host = special(gen, dtype, n, 200)
    if dtype == "f32":
        host[3::7] = 1.0  # (2^100 times the weights leaves fp32)
    if dtype == "bf16":
        host[3::7] = 2.0 ** -119  # (the smallest magnitude that is no zero)
    y = linear8_case(ops, dp, dtype, "none", n, 200, 50, host=host)
    bad = ~torch.isfinite(host).all(1)
    assert torch.equal(torch.isnan(y).all(1).cpu(), bad) and torch.equal(torch.isnan(y).any(1).cpu(), bad)


@pytest.mark.parametrize("n", [2, 50])
def test_the_longest_sums(ops, dp, n):
    """2^17 products of 127 and -128 with the largest magnitude: the sums stay in 32 bits, and are exact."""
    d, o = 2 ** 17, 3
    x = torch.ones(n, d, device="cuda")
    w = torch.full((o, d), 127, dtype=torch.int8, device="cuda")
    w[1] = -128
    w[2, ::2] = -127
    scale, y = torch.ones(o, device="cuda"), torch.empty(n, o, device="cuda")
    ops.linear8(dp.ops.Linear8Shape(n, d, o), x.data_ptr(), w.data_ptr(), scale.data_ptr(), y.data_ptr(),
                stream=stream())
    s = torch.tensor(1 / 127.0).float()
    want = torch.tensor([127.0 * 127 * d, -128.0 * 127 * d, 0.0]) * s
    assert torch.equal(y.cpu(), want.expand(n, o))


def tiles(dp, n, d, o, gate):
    """(tile rows, columns, slices) of a product, from the gated block's plan of as many steps in bf16."""
    k = -(-d // 128) * 64
    plan = dp.ops.GatedShape(n, k, o, 8, dtype="bf16").plan() if gate else \
        dp.ops.GatedShape(n, 8, k, o, dtype="bf16").plan()
    return plan["gate" if gate else "down"]


TILED = [(70, 200, 70), (65, 2060, 33), (260, 40, 6200), (66, 4200, 6200), (700, 500, 900), (3100, 520, 2056),
         (520, 1030, 6200), (3100, 40, 4100), (3100, 200, 2056), (67, 9000, 100)]


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("n,d,o", TILED)
def test_tiles(ops, dp, n, d, o, gate):
    linear8_case(ops, dp, "bf16", "silu", n, d, o, gate, seed=1)


def test_every_tile_shape_is_run(dp):
    """The sizes above meet every tile shape, whole and sliced where a plan slices it."""
    for gate in (False, True):
        seen = {tiles(dp, *s, gate)[:2] for s in TILED + PRODUCTS if s[0] > 64}
        assert seen == {(256, 256), (128, 128), (64, 128), (64, 32)}, (gate, seen)
        assert any(tiles(dp, *s, gate)[2] > 1 for s in TILED + PRODUCTS if s[0] > 64)
        assert any(tiles(dp, *s, gate)[2] == 1 for s in TILED + PRODUCTS if s[0] > 64)


def test_products_past_32_bits(ops, dp):
    """More than 2^32 integers in the rows' 8-bit form, and 2^31 in y's bytes: the first rows and the last."""
    n, d, o = 2 ** 21 + 9, 2064, 520
    x = torch.empty(n, d, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator().manual_seed(1)
    ends = torch.randn(32, d, generator=gen).bfloat16()
    x.fill_(1.0)
    x[:16], x[-16:] = ends[:16].cuda(), ends[16:].cuda()
    w, ws = weights(gen, o, d)
    gw, gs, y = w.cuda(), ws.cuda(), torch.empty(n, o, dtype=torch.bfloat16, device="cuda")
    ops.linear8(dp.ops.Linear8Shape(n, d, o, dtype="bf16"), x.data_ptr(), gw.data_ptr(), gs.data_ptr(), y.data_ptr(),
                stream=stream())
    torch.cuda.synchronize()
    v, b = ref8.linear8("bf16", "none", ends.double(), w[:, :d], ws)
    check(torch.cat([y[:16], y[-16:]]), (v, b), "ends")
    assert bool((y[16:-16] == y[16]).all())


@pytest.mark.parametrize("o", [1, 8])
def test_backward_from_a_checkpoint_past_32_bits(ops, dp, o):
    """More than 2^32 hidden values: dx of the first rows and the last, and a w_down gradient over all."""
    n, d, f = 2 ** 21 + 40, 8, 2072
    gen = torch.Generator().manual_seed(4)
    host = {"wg": rand(gen, "bf16", d, f, d ** -0.5), "wu": rand(gen, "bf16", d, f, d ** -0.5),
            "wd": rand(gen, "bf16", f, o, f ** -0.5)}
    xe, dye = rand(gen, "bf16", 32, d), rand(gen, "bf16", 32, o)
    g = {k: v.cuda() for k, v in host.items()}
    x, dy = (torch.zeros(n, c, dtype=torch.bfloat16, device="cuda") for c in (d, o))
    for m, e in ((x, xe), (dy, dye)):
        m[:16], m[-16:] = e[:16].cuda(), e[16:].cuda()
    dx, dwd = torch.empty_like(x), torch.empty_like(g["wd"])
    kept = kept_of(dp, n, d)
    shape = dp.ops.GatedShape(n, d, f, o, dtype="bf16")
    ops.keep8(x.data_ptr(), kept.data_ptr(), n, d, "bf16", stream=stream())
    ops.gated_backward8(shape, kept.data_ptr(), *(g[k].data_ptr() for k in ("wg", "wu", "wd")), dy.data_ptr(),
                        dx.data_ptr(), d_dw_down=dwd.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    # (the rows between are zeros, whose gradients are: sums over the 32 rows, and over many zeros)
    want = ref.gated("bf16", "silu", ref8.restored(xe.double()), *(host[k].double() for k in ("wg", "wu", "wd")),
                     dye.double())
    check(torch.cat([dx[:16], dx[-16:]]), want["dx"], "dx")
    check(dwd, want["dwd"], "dwd")
    assert bool((dx[16:-16] == 0).all())


def test_restored_past_the_caches(ops, dp):
    """Outputs of over 192 MB are stored in another way."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    for dtype, cols in (("bf16", 1043), ("f32", 1040)):
        x = torch.randn(100000, cols, generator=gen, device="cuda").to(ref.TORCH[dtype])
        kept, out, part = kept_of(dp, 100000, cols), torch.empty_like(x), torch.empty(1000, cols, dtype=x.dtype,
                                                                                     device="cuda")
        ops.keep8(x.data_ptr(), kept.data_ptr(), 100000, cols, dtype, stream=stream())
        ops.restore8(kept.data_ptr(), out.data_ptr(), 100000, cols, dtype, stream=stream())
        few = kept_of(dp, 1000, cols)
        for at in (0, 50000, 99000):
            ops.keep8(x[at:].data_ptr(), few.data_ptr(), 1000, cols, dtype, stream=stream())
            ops.restore8(few.data_ptr(), part.data_ptr(), 1000, cols, dtype, stream=stream())
            assert torch.equal(out[at:at + 1000], part)


@pytest.mark.parametrize("pad,skip", [(0, 0), (3, 1)])
@pytest.mark.parametrize("n,d", [(70, 100), (1100, 100), (1030, 500), (300, 520), (8200, 513), (8203, 1024), (1200, 1031),
                                 (70, 2050), (1100, 4099), (70, 8192), (66, 8200), (1100, 9000)])
def test_rows_of_every_length(ops, dp, n, d, pad, skip):
    """Rows quantised by 16 lanes, a wave or a block, ending inside and beyond what these hold."""
    for k, dtype in enumerate(TYPES):
        linear8_case(ops, dp, dtype, ("tanh", "none", "silu")[k], n, d, 9, pad=pad, skip=skip)
