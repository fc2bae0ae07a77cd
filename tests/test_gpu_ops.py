"""The operators of trainable heads on the GPU against 64 bits, element by element within
the bounds of ops_reference.py: odd and small sizes, each type, sizes at the edges of
the tiles, strided and unaligned matrices, sums over long axes, padding ids."""
import math

import pytest
import torch

import ops_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(dp):
    return dp.ops.Operators()


def stream():
    return torch.cuda.current_stream().cuda_stream


def rand(gen, dtype, rows, cols, size=1.0):
    return (torch.randn(rows, cols, generator=gen, dtype=torch.float64) * size).to(ref.TORCH[dtype])


class Mat:
    """A matrix on the GPU, as columns of a wider one (`pad` more elements a row, `skip`
    elements before it) whose other elements are NaN (inputs) or a marker (outputs)."""

    def __init__(self, host=None, shape=None, dtype=None, pad=0, skip=0, fill=float("nan")):
        r, c = host.shape if host is not None else shape
        self.ld = c + pad
        self.buf = torch.full((skip + max(r, 1) * self.ld,), fill,
                              dtype=host.dtype if host is not None else ref.TORCH[dtype], device="cuda")
        self.view = self.buf[skip:].as_strided((r, c), (self.ld, 1))
        if host is not None:
            self.view.copy_(host)
        self.ptr = self.buf.data_ptr() + skip * self.buf.element_size()

    def untouched(self, fill):
        keep = self.buf.clone()
        keep[self.buf.numel() - max(self.view.shape[0], 1) * self.ld:].as_strided(
            self.view.shape, (self.ld, 1)).fill_(fill)
        return bool((keep == fill).all())


def check(got, want, what):
    v, b = want
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    over = ((got - v).abs() - b)
    assert (over <= 0).all(), (what, float(over.max()), float((got - v).abs().max()), float(b.max()))


def gated_case(ops, dp, dtype, act, n, d, f, o, pad=0, skip=0, seed=0, size=1.0):
    gen = torch.Generator().manual_seed(1000 + seed)
    host = {"x": rand(gen, dtype, n, d, size), "wg": rand(gen, dtype, d, f, d ** -0.5),
            "wu": rand(gen, dtype, d, f, d ** -0.5), "wd": rand(gen, dtype, f, o, f ** -0.5),
            "dy": rand(gen, dtype, n, o)}
    m = {k: Mat(v, pad=pad, skip=skip) for k, v in host.items()}
    for k, s in (("y", (n, o)), ("dx", (n, d)), ("dwg", (d, f)), ("dwu", (d, f)), ("dwd", (f, o))):
        m[k] = Mat(shape=s, dtype=dtype, pad=pad, skip=skip, fill=7.0)
    shape = dp.ops.GatedShape(n, d, f, o, dtype=dtype, act=act, ld_x=m["x"].ld, ld_y=m["y"].ld,
                              ld_hidden=m["wg"].ld, ld_down=m["wd"].ld)
    saved = torch.full((shape.saved_bytes() + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    p = {k: v.ptr for k, v in m.items()}
    y0 = Mat(shape=(n, o), dtype=dtype, pad=pad, skip=skip, fill=7.0)
    ops.gated_forward(shape, p["x"], p["wg"], p["wu"], p["wd"], y0.ptr, stream=stream())
    ops.gated_forward(shape, p["x"], p["wg"], p["wu"], p["wd"], p["y"], saved=saved.data_ptr(), stream=stream())
    ops.gated_backward(shape, p["x"], p["wg"], p["wu"], p["wd"], saved.data_ptr(), p["dy"], p["dx"], p["dwg"],
                       p["dwu"], p["dwd"], stream=stream())
    torch.cuda.synchronize()
    # (large ones' 64-bit products on the GPU: plain matrix products of torch)
    at = "cuda" if n * f * max(d, o) > 2e9 else "cpu"
    want = ref.gated(dtype, act, *(host[k].double().to(at) for k in ("x", "wg", "wu", "wd", "dy")))
    for k, (v, b) in want.items():
        check(m[k].view, (v.cpu(), b.cpu()), (k, dtype, act, n, d, f, o))
        assert m[k].untouched(7.0), k
    # (with a workspace grown by the backward or not, kept or not: the same bits)
    assert torch.equal(y0.view, m["y"].view)
    assert bool((saved[shape.saved_bytes():] == 0xA5).all())
    return shape, m, saved


SIZES = [(1, 1, 1, 1), (1, 64, 128, 32), (2, 7, 9, 5), (3, 8, 8, 8), (16, 32, 16, 16), (17, 33, 65, 31),
         (31, 70, 96, 1), (64, 40, 24, 200), (65, 129, 130, 127), (128, 64, 128, 64), (130, 72, 264, 136),
         (257, 100, 60, 260)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,d,f,o", SIZES)
def test_gated_sizes(ops, dp, dtype, n, d, f, o):
    gated_case(ops, dp, dtype, "silu", n, d, f, o, seed=n + d)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9])
@pytest.mark.parametrize("d,f,o", [(200, 300, 100), (1100, 65, 72), (64, 2100, 9)])
def test_gated_few_rows(ops, dp, dtype, n, d, f, o):
    """Up to eight rows (kernels of their own) and nine: several slices, columns that end inside a
    chunk, slices longer than one block's."""
    gated_case(ops, dp, dtype, "gelu", n, d, f, o, seed=n)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad,skip", [(8, 8), (3, 1)])
def test_gated_few_rows_strides(ops, dp, dtype, pad, skip):
    gated_case(ops, dp, dtype, "silu", 3, 130, 203, 77, pad=pad, skip=skip)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,d,f,o", [(9, 24, 8185, 1), (9, 24, 8193, 1), (13, 40, 4100, 2), (300, 40, 2043, 4),
                                     (300, 40, 2056, 3), (3000, 33, 97, 3), (1, 16, 260, 4), (4111, 16, 260, 5)])
def test_gated_few_outputs(ops, dp, dtype, n, d, f, o):
    """Up to four outputs (kernels of their own), five, and where the hidden side is too wide for them:
    odd widths, several groups of columns, slices of one row and of many."""
    gated_case(ops, dp, dtype, "tanh", n, d, f, o, seed=n + o)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("pad,skip", [(8, 8), (3, 1)])
def test_gated_few_outputs_strides(ops, dp, dtype, pad, skip):
    gated_case(ops, dp, dtype, "silu", 70, 33, 131, 3, pad=pad, skip=skip)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("act", ["tanh", "gelu"])
def test_gated_activations(ops, dp, dtype, act):
    gated_case(ops, dp, dtype, act, 70, 48, 80, 24, seed=5, size=3.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("pad,skip", [(8, 0), (8, 8), (3, 0), (0, 1), (5, 3)])
def test_gated_strides(ops, dp, dtype, pad, skip):
    """Columns of wider matrices whose other elements are NaN, aligned and not."""
    gated_case(ops, dp, dtype, "silu", 33, 40, 72, 24, pad=pad, skip=skip, seed=pad)
    gated_case(ops, dp, dtype, "silu", 33, 41, 71, 23, pad=pad, skip=skip, seed=pad)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,d,f,o", [(5000, 70, 96, 1), (9, 1000, 700, 300), (700, 600, 500, 400),
                                     (2100, 300, 520, 264)])
def test_gated_long_axes(ops, dp, dtype, n, d, f, o):
    """Sums over many rows or columns (cut into slices), several tiles each way."""
    gated_case(ops, dp, dtype, "silu", n, d, f, o, seed=n)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,d,f,o", [(9001, 515, 1031, 520), (12300, 1601, 242, 250), (8201, 1031, 4105, 2060),
                                     (4101, 64, 8201, 4100)])
def test_gated_large_tiles(ops, dp, dtype, n, d, f, o):
    """Each tile shape in every product that takes it, with edges inside its tiles."""
    gated_case(ops, dp, dtype, "silu", n, d, f, o, seed=n)


def test_gated_many_tiles(ops, dp):
    """Enough tiles for the largest tile shape: rows against 64 bits at random."""
    gen = torch.Generator().manual_seed(3)
    n, d, f, o = 8200, 264, 2056, 1032
    host = [rand(gen, "bf16", *s) for s in ((n, d), (d, f), (d, f), (f, o))]
    host[1] *= d ** -0.5
    host[2] *= d ** -0.5
    host[3] *= f ** -0.5
    m = [Mat(h) for h in host]
    y = Mat(shape=(n, o), dtype="bf16")
    shape = dp.ops.GatedShape(n, d, f, o, dtype="bf16", act="silu")
    ops.gated_forward(shape, *(k.ptr for k in m), y.ptr, stream=stream())
    rows = torch.randperm(n, generator=gen)[:200]
    rows[:2] = torch.tensor([0, n - 1])
    want = ref.gated("bf16", "silu", host[0][rows].double(), *(h.double() for h in host[1:]))["y"]
    check(y.view.cpu()[rows], want, "y")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gated_parts_of_the_backward(ops, dp, dtype):
    """Outputs that are not asked for are not needed by the others."""
    shape, m, saved = gated_case(ops, dp, dtype, "silu", 50, 24, 40, 16)
    p = {k: v.ptr for k, v in m.items()}
    whole = {k: m[k].view.clone() for k in ("dx", "dwg", "dwu", "dwd")}
    for names in (["dx"], ["dwd"], ["dwg", "dwu"], ["dx", "dwd"], []):
        for k in whole:
            m[k].view.fill_(7.0)
        a = [p[k] if k in names else 0 for k in ("dx", "dwg", "dwu", "dwd")]
        ops.gated_backward(shape, p["x"], p["wg"], p["wu"], p["wd"], saved.data_ptr(), p["dy"], *a, stream=stream())
        for k in whole:
            assert torch.equal(m[k].view, whole[k] if k in names else torch.full_like(whole[k], 7.0)), (names, k)


def test_gated_side_by_side_weights(ops, dp):
    """Gate and up as the halves of one matrix, and so their gradients."""
    gen = torch.Generator().manual_seed(8)
    n, d, f, o = 40, 32, 48, 16
    host = [rand(gen, "bf16", n, d), rand(gen, "bf16", d, 2 * f, d ** -0.5), rand(gen, "bf16", f, o, f ** -0.5),
            rand(gen, "bf16", n, o)]
    x, w, wd, dy = (h.cuda() for h in host)
    y, dx, dw, dwd = (torch.empty_like(t) for t in (dy, x, w, wd))
    shape = dp.ops.GatedShape(n, d, f, o, dtype="bf16", act="silu", ld_hidden=2 * f)
    saved = torch.empty(shape.saved_bytes(), dtype=torch.uint8, device="cuda")
    wp, gp = w.data_ptr(), dw.data_ptr()
    ops.gated_forward(shape, x.data_ptr(), wp, wp + 2 * f, wd.data_ptr(), y.data_ptr(), saved=saved.data_ptr(),
                      stream=stream())
    ops.gated_backward(shape, x.data_ptr(), wp, wp + 2 * f, wd.data_ptr(), saved.data_ptr(), dy.data_ptr(),
                       dx.data_ptr(), gp, gp + 2 * f, dwd.data_ptr(), stream=stream())
    h = [t.double() for t in host]
    want = ref.gated("bf16", "silu", h[0], h[1][:, :f], h[1][:, f:], h[2], h[3])
    for k, got in (("y", y), ("dx", dx), ("dwg", dw[:, :f]), ("dwu", dw[:, f:]), ("dwd", dwd)):
        check(got, want[k], k)


def test_gated_against_differences(ops, dp):
    """Directional derivatives of sum(dy * y) by central differences of the forward on the
    GPU, against the backward's. Allowed: the differences' own truncation (from the
    formula in 64 bits) and the bounds of the forward's and the backward's values."""
    gen = torch.Generator().manual_seed(21)
    n, d, f, o, eps = 12, 24, 40, 8, 2.0 ** -5
    names = ("x", "wg", "wu", "wd")
    base = dict(zip(names, (rand(gen, "f32", n, d), rand(gen, "f32", d, f, d ** -0.5),
                            rand(gen, "f32", d, f, d ** -0.5), rand(gen, "f32", f, o, f ** -0.5))))
    dy = rand(gen, "f32", n, o)
    shape = dp.ops.GatedShape(n, d, f, o, dtype="f32", act="gelu")
    saved = torch.empty(shape.saved_bytes(), dtype=torch.uint8, device="cuda")

    def forward(v, keep=0):
        dev = [v[k].cuda() for k in names]
        y = torch.empty(n, o, device="cuda")
        ops.gated_forward(shape, *(t.data_ptr() for t in dev), y.data_ptr(), saved=keep, stream=stream())
        torch.cuda.synchronize()
        return dev, y.double().cpu()

    dev, _ = forward(base, saved.data_ptr())
    grads = [torch.empty_like(t) for t in dev]
    ddy = dy.cuda()
    ops.gated_backward(shape, *(t.data_ptr() for t in dev), saved.data_ptr(), ddy.data_ptr(),
                       *(t.data_ptr() for t in grads), stream=stream())
    torch.cuda.synchronize()
    bounds = ref.gated("f32", "gelu", *(base[k].double() for k in names), dy.double())
    for k, got, out in zip(names, grads, ("dx", "dwg", "dwu", "dwd")):
        way = torch.randn(base[k].shape, generator=gen)
        sides, exact, noise = [], [], 0.0
        for s in (eps, -eps):
            v = dict(base, **{k: base[k] + s * way})
            sides.append((forward(v)[1] * dy.double()).sum())
            y, b = ref.gated("f32", "gelu", *(v[q].double() for q in names))["y"]
            exact.append((y * dy.double()).sum())
            noise += float((b * dy.abs().double()).sum())
        # the steps that 32 bits really took
        step = ((base[k] + eps * way).double() - (base[k] - eps * way).double()) / (2 * eps)
        slope64 = float((bounds[out][0] * step).sum())
        truncation = abs(float(exact[0] - exact[1]) / (2 * eps) - slope64)
        slack = float((bounds[out][1] * step.abs()).sum())
        diff = float(sides[0] - sides[1]) / (2 * eps)
        slope = float((got.double().cpu() * step).sum())
        allowed = truncation + noise / (2 * eps) + slack
        assert abs(diff - slope) <= allowed, (k, diff, slope)
        assert abs(slope64) > 2 * allowed, k  # (a gradient half as large, or of the other sign, is told)


def test_gated_no_rows(ops, dp):
    shape = dp.ops.GatedShape(0, 8, 16, 4, dtype="bf16", act="silu", ld_hidden=20)
    assert shape.saved_bytes() == 0
    ops.gated_forward(shape, 0, 0, 0, 0, 0, stream=stream())
    dwg, dwu = (torch.full((8, 20), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    dwd = torch.full((16, 4), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.gated_backward(shape, 0, 0, 0, 0, 0, 0, 0, dwg.data_ptr(), dwu.data_ptr(), dwd.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    for t in (dwg, dwu):
        assert not t[:, :16].any() and bool((t[:, 16:] == 7).all())
    assert not dwd.any()


def test_gated_nan_stays_in_its_row(ops, dp):
    """A row of NaN (an atom left out) spoils its own outputs alone, and the weights' gradients."""
    n, d, f, o = 40, 24, 48, 16
    gen = torch.Generator().manual_seed(4)
    x = rand(gen, "bf16", n, d)
    w = [rand(gen, "bf16", d, f, .2).cuda(), rand(gen, "bf16", d, f, .2).cuda(), rand(gen, "bf16", f, o, .2).cuda()]
    shape = dp.ops.GatedShape(n, d, f, o, dtype="bf16")
    ys = []
    for bad in (False, True):
        xd = x.clone()
        if bad:
            xd[17] = float("nan")
        xd = xd.cuda()
        y = torch.empty(n, o, dtype=torch.bfloat16, device="cuda")
        ops.gated_forward(shape, xd.data_ptr(), *(t.data_ptr() for t in w), y.data_ptr(), stream=stream())
        ys.append(y.cpu())
    keep = torch.arange(n) != 17
    assert torch.equal(ys[0][keep], ys[1][keep]) and torch.isnan(ys[1][17]).all()


def test_gated_streams_and_graph(ops, dp):
    """Calls on two streams at once, and replays of a captured call between eager ones."""
    n, d, f, o = 200, 64, 96, 32
    gen = torch.Generator().manual_seed(6)
    w = [rand(gen, "bf16", d, f, .2).cuda(), rand(gen, "bf16", d, f, .2).cuda(), rand(gen, "bf16", f, o, .2).cuda()]
    shape = dp.ops.GatedShape(n, d, f, o, dtype="bf16")
    xs = [rand(gen, "bf16", n, d).cuda() for _ in range(3)]
    one = dp.ops.Operators()

    def call(x, y, st):
        one.gated_forward(shape, x.data_ptr(), *(t.data_ptr() for t in w), y.data_ptr(), stream=st)

    want = []
    for x in xs:
        y = torch.empty(n, o, dtype=torch.bfloat16, device="cuda")
        call(x, y, stream())
        want.append(y)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    ys = [torch.zeros_like(want[0]) for _ in range(6)]
    torch.cuda.synchronize()
    for k in range(6):
        call(xs[k % 3], ys[k], streams[k % 2].cuda_stream)
    torch.cuda.synchronize()
    for k in range(6):
        assert torch.equal(ys[k], want[k % 3])

    fresh = dp.ops.Operators()
    st = torch.cuda.Stream()
    x, y = xs[0].clone(), torch.zeros_like(want[0])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()

    def captured():
        fresh.gated_forward(shape, x.data_ptr(), *(t.data_ptr() for t in w), y.data_ptr(),
                            stream=torch.cuda.current_stream().cuda_stream)

    with torch.cuda.stream(st):
        captured()  # the workspace of this stream
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        captured()
    for k in (1, 2, 0):
        x.copy_(xs[k])
        y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[k])
        again = torch.zeros_like(y)
        call(xs[k], again, stream())  # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(again, want[k])


# ---- embedding -------------------------------------------------------------------------
def ids_of(gen, n, vocab, kind):
    if kind == "skewed":  # one id holds most rows
        ids = torch.randint(0, vocab, (n,), generator=gen)
        ids[torch.rand(n, generator=gen) < 0.7] = vocab // 2
    elif kind == "one":
        ids = torch.full((n,), vocab - 1)
    else:
        ids = torch.randint(0, vocab, (n,), generator=gen)
    out = torch.rand(n, generator=gen)
    ids[out < 0.05] = -1
    ids[out > 0.97] = vocab
    if n > 3:
        ids[1], ids[2] = -2 ** 31, 2 ** 31 - 1
    return ids.int()


EMBED = [(1, 1, 1), (5, 2, 8), (192, 2, 8), (33, 300, 7), (257, 118, 64), (1000, 3, 130), (2049, 70000, 16),
         (4100, 257, 33), (3000, 50, 520)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,vocab,width", [(8192, 70001, 12), (8193, 70001, 12), (20000, 300, 40),
                                           (140000, 20000, 5), (65, 20000, 9)])
def test_embed_gradient_forms(ops, dtype, n, vocab, width):
    """Rows on both sides of each form of the sort: one block, tiles with their own starts,
    tiles with scanned ones; ids of more than 16 bits; a table of few and of many rows."""
    gen = torch.Generator().manual_seed(n)
    ids = ids_of(gen, n, vocab, "skewed")
    dout = rand(gen, dtype, n, width)
    dt = Mat(shape=(vocab, width), dtype=dtype, fill=7.0)
    d_ids, d_dout = ids.cuda(), dout.cuda()
    for _ in range(2):  # (the second finds what the first left in the workspace)
        ops.embed_grad(d_ids.data_ptr(), d_dout.data_ptr(), dt.ptr, n, vocab, width, dtype, stream=stream())
        torch.cuda.synchronize()
        check(dt.view, ref.embed_grad(dtype, ids, dout.double(), vocab, 1.0), "embed_grad")
        ids = ids.flip(0)
        d_ids = ids.cuda()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,vocab,width", EMBED)
@pytest.mark.parametrize("kind", ["even", "skewed", "one"])
def test_embed_and_gradient(ops, dtype, n, vocab, width, kind):
    gen = torch.Generator().manual_seed(n + vocab)
    ids = ids_of(gen, n, vocab, kind)
    table, dout = rand(gen, dtype, vocab, width), rand(gen, dtype, n, width)
    d_ids = ids.cuda()
    for pad, skip in ((0, 0), (3, 1), (8, 4)):
        t, g = Mat(table, pad=pad, skip=skip), Mat(dout, pad=pad, skip=skip)
        out = Mat(shape=(n, width), dtype=dtype, pad=pad, skip=skip, fill=7.0)
        dt = Mat(shape=(vocab, width), dtype=dtype, pad=pad, skip=skip, fill=7.0)
        ops.embed(d_ids.data_ptr(), t.ptr, out.ptr, n, vocab, width, dtype, scale=0.625, ld_table=t.ld,
                  ld_out=out.ld, stream=stream())
        ops.embed_grad(d_ids.data_ptr(), g.ptr, dt.ptr, n, vocab, width, dtype, scale=0.625, ld_dout=g.ld,
                       ld_dtable=dt.ld, stream=stream())
        torch.cuda.synchronize()
        check(out.view, ref.embed(dtype, ids, table.double(), 0.625), "embed")
        check(dt.view, ref.embed_grad(dtype, ids, dout.double(), vocab, 0.625), "embed_grad")
        assert out.untouched(7.0) and dt.untouched(7.0)


def test_embed_gradient_repeats_and_order(ops):
    """The same bits whenever it is called, and sums that a permutation of the other ids' rows
    does not change."""
    gen = torch.Generator().manual_seed(2)
    n, vocab, width = 20000, 40, 96
    ids = ids_of(gen, n, vocab, "skewed").cuda()
    dout = rand(gen, "f32", n, width).cuda()
    outs = []
    for _ in range(3):
        dt = torch.empty(vocab, width, device="cuda")
        ops.embed_grad(ids.data_ptr(), dout.data_ptr(), dt.data_ptr(), n, vocab, width, stream=stream())
        outs.append(dt)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("repeat", [1, 9])
@pytest.mark.parametrize("width", [3, 520])
@pytest.mark.parametrize("empty", [2500, 9000, 20000])
def test_embed_gradient_lengths_of_runs(ops, repeat, width, empty):
    """Runs around one window and the length from which windows sum them, at every offset to
    the windows (lead), up to the last position; exact, on small whole numbers. In one block of the sort and in
    tiles, with one table row a wave, four and eight."""
    gen = torch.Generator().manual_seed(11)
    lengths = [31, 32, 33, 63, 64, 65, 1, 66, 0, 95, 96, 97, 2, 127, 128, 129, 64, 65] * repeat
    vocab = 3 * len(lengths) + empty
    for lead in (0, 1, 30, 31, 32, 33):
        counts = torch.tensor([lead] + lengths)
        ids = torch.repeat_interleave(3 * torch.arange(len(counts)), counts)
        ids = ids[torch.randperm(len(ids), generator=gen)].int().cuda()
        dout = torch.randint(-8, 9, (len(ids), width), generator=gen).float().cuda()
        dt = torch.full((vocab, width), 7.0, device="cuda")
        ops.embed_grad(ids.data_ptr(), dout.data_ptr(), dt.data_ptr(), len(ids), vocab, width, stream=stream())
        want = torch.zeros(vocab, width, dtype=torch.float64).index_add_(0, ids.cpu().long(), dout.double().cpu())
        torch.cuda.synchronize()
        assert torch.equal(dt.double().cpu(), want), lead


def test_embed_gradient_is_the_lookup_transposed(ops):
    """<lookup(table), w> = <table, gradient(w)>, exactly, on small whole numbers."""
    gen = torch.Generator().manual_seed(9)
    n, vocab, width = 5000, 300, 40
    ids = ids_of(gen, n, vocab, "skewed").cuda()
    table = torch.randint(-4, 5, (vocab, width), generator=gen).float().cuda()
    w = torch.randint(-4, 5, (n, width), generator=gen).float().cuda()
    out, dt = torch.empty(n, width, device="cuda"), torch.empty(vocab, width, device="cuda")
    ops.embed(ids.data_ptr(), table.data_ptr(), out.data_ptr(), n, vocab, width, scale=2.0, stream=stream())
    ops.embed_grad(ids.data_ptr(), w.data_ptr(), dt.data_ptr(), n, vocab, width, scale=2.0, stream=stream())
    assert float((out.double() * w.double()).sum()) == float((table.double() * dt.double()).sum())


def test_embed_nothing(ops):
    dt = torch.full((5, 9), 7.0, device="cuda")
    ops.embed(0, 0, dt.data_ptr(), 0, 5, 9, stream=stream())
    ops.embed_grad(0, 0, dt.data_ptr(), 0, 5, 8, ld_dtable=9, stream=stream())
    torch.cuda.synchronize()
    assert not dt[:, :8].any() and bool((dt[:, 8] == 7).all())
    # ids that are all outside the table
    ids = torch.full((70,), -1, dtype=torch.int32, device="cuda")
    g = torch.full((70, 8), float("nan"), device="cuda")
    ops.embed_grad(ids.data_ptr(), g.data_ptr(), dt.data_ptr(), 70, 5, 8, ld_dtable=9, stream=stream())
    torch.cuda.synchronize()
    assert not dt[:, :8].any()


# ---- offsets past 32 bits ----------------------------------------------------------------
def test_offsets_past_32_bits(ops, dp):
    """Rows that lie more than 2^32 elements into a matrix."""
    gen = torch.Generator().manual_seed(12)
    n, ld, d, f, o = (1 << 20) + 300, 4112, 16, 24, 8
    x = torch.zeros(n, ld, dtype=torch.bfloat16, device="cuda")
    last = rand(gen, "bf16", 300, d)
    x[-300:, :d] = last.cuda()
    w = [rand(gen, "bf16", d, f, .25), rand(gen, "bf16", d, f, .25), rand(gen, "bf16", f, o, .2)]
    y = torch.full((n, o), 7.0, dtype=torch.bfloat16, device="cuda")
    shape = dp.ops.GatedShape(n, d, f, o, dtype="bf16", ld_x=ld)
    dw = [t.cuda() for t in w]
    ops.gated_forward(shape, x.data_ptr(), *(t.data_ptr() for t in dw), y.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    check(y[-300:], ref.gated("bf16", "silu", last.double(), *(t.double() for t in w))["y"], "y")
    assert not y[:-300].any()
    # the same matrix as a table: its last rows, and their gradient
    ids = torch.arange(n - 300, n, dtype=torch.int32)
    out = torch.empty(300, d, dtype=torch.bfloat16, device="cuda")
    d_ids = ids.cuda()
    ops.embed(d_ids.data_ptr(), x.data_ptr(), out.data_ptr(), 300, n, d, "bf16", ld_table=ld, stream=stream())
    assert torch.equal(out.cpu(), last)
    x[-300:, :d] = 0
    ops.embed_grad(d_ids.data_ptr(), out.data_ptr(), x.data_ptr(), 300, n, d, "bf16", ld_dtable=ld, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(x[-300:, :d].cpu(), last)


def test_example_learns(dp):
    """The head of examples/train_head.py learns its targets: half of their variance within 30 steps."""
    import importlib.util
    import os

    from _pkg import ROOT
    spec = importlib.util.spec_from_file_location("train_head", os.path.join(ROOT, "examples", "train_head.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    losses = mod.train(dp, steps=30, cells=2)
    assert all(math.isfinite(v) for v in losses) and losses[-1] < 0.5 * losses[0]


# ---- refusals ---------------------------------------------------------------------------
def test_refusals(ops, dp):
    S = dp.ops.GatedShape
    p = torch.empty(4096, device="cuda").data_ptr()
    bad = [S(-1, 8, 8, 8), S(4, 0, 8, 8), S(4, 8, 0, 8), S(4, 8, 8, 0), S(4, 8, 8, 8, dtype="f64"),
           S(4, 8, 8, 8, act="relu"), S(4, 8, 8, 8, ld_x=7), S(4, 8, 8, 8, ld_y=7), S(4, 8, 8, 8, ld_hidden=7),
           S(4, 8, 8, 8, ld_down=7), S(2 ** 40, 8, 8, 8), S(4, 2 ** 21, 8, 8), S(4, 8, 8, 8, ld_x=2 ** 40)]
    for s in bad:
        assert s.saved_bytes() == 0
        with pytest.raises(dp.DeepmdException):
            ops.gated_forward(s, p, p, p, p, p)
        with pytest.raises(dp.DeepmdException):
            ops.gated_backward(s, p, p, p, p, p, p, p)
    good = S(4, 8, 8, 8)
    for k in range(5):
        with pytest.raises(dp.DeepmdException, match="null"):
            ops.gated_forward(good, *(0 if q == k else p for q in range(5)))
    with pytest.raises(dp.DeepmdException, match="aligned"):
        ops.gated_forward(good, p, p, p, p, p, saved=p + 4)
    with pytest.raises(dp.DeepmdException, match="both"):
        ops.gated_backward(good, p, p, p, p, p, p, p, p, 0, p)
    for args in ((-1, 4, 8), (4, 0, 8), (4, 4, 0), (2 ** 40, 4, 8)):
        with pytest.raises(dp.DeepmdException):
            ops.embed(p, p, p, *args)
        with pytest.raises(dp.DeepmdException):
            ops.embed_grad(p, p, p, *args)
    for kw in (dict(ld_table=7), dict(ld_out=7), dict(dtype="f64")):
        with pytest.raises(dp.DeepmdException):
            ops.embed(p, p, p, 4, 4, 8, **kw)
    for k in range(3):
        with pytest.raises(dp.DeepmdException, match="null"):
            ops.embed(*(0 if q == k else p for q in range(3)), 4, 4, 8)
        with pytest.raises(dp.DeepmdException, match="null"):
            ops.embed_grad(*(0 if q == k else p for q in range(3)), 4, 4, 8)


def test_no_memory_is_an_error(dp):
    """A workspace that no card holds is an error before anything is launched, and the next call works."""
    one = dp.ops.Operators()
    p = torch.zeros(4096, device="cuda").data_ptr()
    with pytest.raises(dp.DeepmdException, match="HIP error"):
        one.gated_forward(dp.ops.GatedShape(2 ** 30, 8, 2 ** 20, 8), p, p, p, p, p)
    with pytest.raises(dp.DeepmdException, match="HIP error"):
        one.embed_grad(p, p, p, 2 ** 30, 2 ** 30, 2 ** 20)
    gated_case(one, dp, "f32", "silu", 20, 8, 16, 8)
    assert one.device_bytes() > 0


def test_capture_needs_a_workspace(dp):
    """A call whose workspace would have to grow inside a capture is refused, and the capture lives on."""
    one = dp.ops.Operators()
    s = dp.ops.GatedShape(4, 8, 8, 8)
    t = torch.zeros(4096, device="cuda")
    p = t.data_ptr()
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        with pytest.raises(dp.DeepmdException, match="capture"):
            one.gated_forward(s, p, p + 1024, p + 2048, p + 4096, p + 8192, stream=st.cuda_stream)
        t.add_(1.0)
    graph.replay()
    torch.cuda.synchronize()
    assert bool((t == 1.0).all()) and math.isfinite(float(t.sum()))
