"""Group norm with an activation, forward and backward, on the GPU against 64 bits within the bounds of
ops8_reference.py: frames of one row and of many, ragged and empty ones, groups of one channel and of all, odd
sizes, strides, large means, rows that belong to no frame."""
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


def norm_case(ops, dp, dtype, act, rows, ch, groups, frames=1, lengths=None, first=0, kept=False, pad=0, skip=0,
              affine=True, which=("dx", "dgamma", "dbeta"), shift=0.5, size=1.0, eps=1e-5, stats=True, seed=0, at="cpu"):
    gen = torch.Generator().manual_seed(rows + ch + groups + seed)
    t = ref.TORCH[dtype]
    host = {"x": ((torch.randn(rows, ch, generator=gen, dtype=torch.float64) + shift) * size).to(t),
            "dy": rand(gen, dtype, rows, ch)}
    gamma, beta = rand(gen, dtype, 1, ch), rand(gen, dtype, 1, ch)
    starts = None
    if lengths is None:
        each = rows // frames
        parts = [(f * each, each) for f in range(frames)]
    else:
        frames = len(lengths)
        ends = [first]
        for n in lengths:
            ends.append(ends[-1] + n)
        parts = list(zip(ends[:-1], lengths))
        starts = torch.tensor(ends, dtype=torch.int32, device="cuda")
    m = {k: Mat(v, pad=pad, skip=skip) for k, v in host.items()}
    for k in ("y", "dx"):
        m[k] = Mat(shape=(rows, ch), dtype=dtype, pad=pad, skip=skip, fill=7.0)
    for k in ("dgamma", "dbeta"):
        m[k] = Mat(shape=(1, ch), dtype=dtype, skip=skip, fill=7.0)
    g, b = (Mat(v, skip=skip) for v in (gamma, beta))
    shape = dp.ops.NormShape(rows, ch, groups, frames=frames, dtype=dtype, act=act, eps=eps, ld_x=m["x"].ld,
                             ld_y=m["y"].ld)
    st = torch.full((frames * groups * 2 + 4,), 7.0, device="cuda")
    sp = 0 if starts is None else starts.data_ptr()
    gp, bp = (g.ptr, b.ptr) if affine else (0, 0)
    if not stats:
        ops.group_norm(shape, m["x"].ptr, gp, bp, m["y"].ptr, starts=sp, stream=stream())
        alone = m["y"].view.clone()
        m["y"].view.fill_(7.0)
    ops.group_norm(shape, m["x"].ptr, gp, bp, m["y"].ptr, stats=st.data_ptr(), starts=sp, stream=stream())
    kp, xp = 0, m["x"].ptr
    if kept:
        buf = torch.empty(dp.ops.keep8_bytes(rows, ch), dtype=torch.uint8, device="cuda")
        ops.keep8(xp, buf.data_ptr(), rows, ch, dtype, ld_x=m["x"].ld, stream=stream())
        kp, xp = buf.data_ptr(), 0
    given = [m[k].ptr if k in which else 0 for k in ("dx", "dgamma", "dbeta")]
    ops.group_norm_grad(shape, xp, gp, bp, st.data_ptr(), m["dy"].ptr, *given, kept=kp, starts=sp, stream=stream())
    torch.cuda.synchronize()
    if not stats:
        assert torch.equal(alone, m["y"].view)
    one, zero = torch.ones(ch, dtype=torch.float64), torch.zeros(ch, dtype=torch.float64)
    args = [host["x"].double(), gamma[0].double() if affine else one, beta[0].double() if affine else zero]
    back = ref8.restored(host["x"].double()).to(at) if kept else None
    want = ref8.norm(dtype, act, *(v.to(at) for v in args), parts, groups, eps, host["dy"].double().to(at), back)
    want = {k: (v.cpu(), b.cpu()) for k, (v, b) in want.items()}
    what = (dtype, act, rows, ch, groups, frames, kept)
    check(st[:-4].reshape(frames, groups, 2), want["stats"], ("stats",) + what)
    assert bool((st[-4:] == 7.0).all())
    inside = ~torch.isnan(want["y"][0])
    for k in ("y", "dx"):
        v, bound = want[k]
        if k == "dx" and k not in which:
            assert bool((m[k].view == 7.0).all())
        else:
            check(m[k].view.cpu()[inside], (v[inside], bound[inside]), (k,) + what)
            assert bool((m[k].view.cpu()[~inside] == 7.0).all()), k  # (rows of no frame)
        assert m[k].untouched(7.0), k
    for k in ("dgamma", "dbeta"):
        if k in which:
            check(m[k].view[0], want[k], (k,) + what)
        else:
            assert bool((m[k].view == 7.0).all())
        assert m[k].untouched(7.0), k
    return {k: m[k].view.clone() for k in ("y", "dx", "dgamma", "dbeta")}


# rows, channels, groups, frames: rows by themselves (16, 64, 256 threads a row), frames of a few rows, one frame
SIZES = [(1, 8, 1, 1), (1, 1, 1, 1), (5, 16, 2, 5), (70, 70, 7, 70), (33, 240, 1, 33), (64, 512, 512, 64),
         (100, 2048, 32, 100), (7, 4096, 16, 7), (3, 7000, 7, 3), (40, 30, 3, 8), (192, 1600, 100, 1),
         (96, 70, 1, 4), (300, 64, 64, 3), (512, 24, 2, 2), (1000, 240, 30, 10), (2000, 48, 6, 1),
         (2100, 130, 13, 3), (50, 5000, 2, 5), (9, 12000, 3, 9)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,ch,groups,frames", SIZES)
def test_sizes(ops, dp, dtype, rows, ch, groups, frames):
    act = ("none", "silu", "tanh", "gelu")[(rows + ch) % 4]
    first = norm_case(ops, dp, dtype, act, rows, ch, groups, frames)
    again = norm_case(ops, dp, dtype, act, rows, ch, groups, frames, stats=False)
    assert all(torch.equal(first[k], again[k]) for k in first)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,ch,groups,frames", [s for s in SIZES if s[0] > 1])
def test_from_a_checkpoint(ops, dp, dtype, rows, ch, groups, frames):
    norm_case(ops, dp, dtype, "silu", rows, ch, groups, frames, kept=True, eps=1e-3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("ch,groups", [(64, 8), (70, 7), (33, 1), (1600, 100), (4200, 2)])
@pytest.mark.parametrize("lengths,rows,first", [([5, 0, 17, 1, 40], 70, 0), ([0, 0, 0], 9, 0), ([30], 30, 0),
                                                ([1, 1, 1, 2], 8, 2), ([300, 0, 3], 310, 5)])
def test_ragged(ops, dp, dtype, kept, ch, groups, lengths, rows, first):
    """Frames of unequal lengths, empty ones, rows before the first and behind the last."""
    norm_case(ops, dp, dtype, "gelu", rows, ch, groups, lengths=lengths, first=first, kept=kept, eps=1e-3)


def test_starts_beyond_the_rows(ops, dp):
    """Starts outside the rows are cut off: nothing beyond the arrays is touched."""
    rows, ch = 20, 32
    x = torch.randn(rows, ch, device="cuda")
    for starts, frames in (([-5, 4, 90], [(0, 4), (4, 16)]), ([25, 30, 40], []), ([8, 3, 10], [(3, 7)])):
        s = torch.tensor(starts, dtype=torch.int32, device="cuda")
        buf = torch.full((3, rows, ch), 7.0, device="cuda")
        shape = dp.ops.NormShape(rows, ch, 4, frames=2, eps=1e-3)
        ops.group_norm(shape, x.data_ptr(), 0, 0, buf[1].data_ptr(), starts=s.data_ptr(), stream=stream())
        want = buf.clone().fill_(7.0)
        for f, n in frames:
            a = x[f:f + n].double().reshape(n, 4, 8)
            m = a.mean((0, 2), keepdim=True)
            r = ((a - m).square().mean((0, 2), keepdim=True) + 1e-3) ** -0.5
            want[1, f:f + n] = ((a - m) * r).reshape(n, ch).float()
        assert torch.allclose(buf, want, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,skip", [(8, 8), (3, 1), (1, 0)])
@pytest.mark.parametrize("rows,ch,groups,frames", [(20, 64, 4, 20), (30, 70, 7, 3), (600, 40, 1, 1), (12, 4400, 2, 3)])
def test_strides(ops, dp, dtype, pad, skip, rows, ch, groups, frames):
    norm_case(ops, dp, dtype, "silu", rows, ch, groups, frames, pad=pad, skip=skip)
    norm_case(ops, dp, dtype, "silu", rows, ch, groups, frames, pad=pad, skip=skip, kept=True, eps=1e-3)


@pytest.mark.parametrize("frames", [60, 6, 1])
@pytest.mark.parametrize("which", [("dx",), ("dgamma",), ("dbeta",), ("dgamma", "dbeta"), ()])
@pytest.mark.parametrize("ch,groups", [(48, 4), (4400, 2)])
def test_some_outputs_and_no_affine(ops, dp, frames, which, ch, groups):
    norm_case(ops, dp, "f32", "tanh", 60, ch, groups, frames, which=which)
    norm_case(ops, dp, "bf16", "tanh", 60, ch, groups, frames, which=which, affine=False)


@pytest.mark.parametrize("frames", [64, 4, 1])
@pytest.mark.parametrize("shift,size", [(1000.0, 1.0), (0.0, 1e-12), (3.0, 1e12), (1.0, 2.0 ** -60)])
def test_means_and_scales(ops, dp, frames, shift, size):
    """Means far larger than the deviations, and values whose squares leave fp32's range or almost do."""
    norm_case(ops, dp, "f32", "none", 256, 64, 4, frames, shift=shift, size=size,
              eps=1e-5 if size == 1.0 else 0.0)


@pytest.mark.parametrize("frames", [64, 4, 1])
def test_equal_values(ops, dp, frames):
    """A group without any deviation: y is act(beta), and eps decides."""
    x = torch.full((64, 32), 3.25, device="cuda")
    y, stats = torch.empty_like(x), torch.empty(frames, 4, 2, device="cuda")
    shape = dp.ops.NormShape(64, 32, 4, frames=frames, eps=1e-4)
    ops.group_norm(shape, x.data_ptr(), 0, 0, y.data_ptr(), stats=stats.data_ptr(), stream=stream())
    assert bool((y == 0).all()) and bool((stats[..., 0] == 3.25).all())
    assert torch.allclose(stats[..., 1], torch.tensor(100.0, device="cuda"), rtol=1e-6)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("frames", [64, 4, 1])
def test_values_that_are_not_finite(ops, dp, frames, bad):
    """They make their own frame's group NaN, and nothing else."""
    x = torch.randn(64, 32, device="cuda")
    x[40, 9] = bad
    y = torch.empty_like(x)
    shape = dp.ops.NormShape(64, 32, 4, frames=frames, act="silu")
    ops.group_norm(shape, x.data_ptr(), 0, 0, y.data_ptr(), stream=stream())
    each, want = 64 // frames, torch.zeros(64, 32, dtype=torch.bool)
    f = 40 // each
    want[f * each:(f + 1) * each, 8:16] = True
    assert torch.equal(torch.isnan(y).cpu(), want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,ch,groups,frames", [(20000, 64, 4, 1), (9000, 256, 16, 2), (30000, 16, 16, 30000)])
def test_long(ops, dp, dtype, rows, ch, groups, frames):
    norm_case(ops, dp, dtype, "silu", rows, ch, groups, frames)
    norm_case(ops, dp, dtype, "silu", rows, ch, groups, frames, kept=True)


@pytest.mark.parametrize("frames,lengths", [(3000, None), (None, [1] * 200 + [7] * 300 + [0] * 100 + [50] * 14)])
def test_many_frames(ops, dp, frames, lengths):
    """More frames than blocks."""
    norm_case(ops, dp, "f32", "silu", 3000, 40, 2, frames or 1, lengths=lengths, eps=1e-3)
    norm_case(ops, dp, "f32", "silu", 3000, 1040, 1, frames or 1, lengths=lengths, eps=1e-3)


@pytest.mark.parametrize("frames", [40, 4, 1])
def test_against_differences(ops, dp, frames):
    """dx of one output's sum against differences of the forward in fp64."""
    rows, ch, groups, h = 40, 12, 3, 1e-4
    gen = torch.Generator().manual_seed(2)
    x, dy = (torch.randn(rows, ch, generator=gen) for _ in range(2))
    gx, gdy = x.cuda(), dy.cuda()
    y, dx, stats = torch.empty_like(gx), torch.empty_like(gx), torch.empty(frames, groups, 2, device="cuda")
    shape = dp.ops.NormShape(rows, ch, groups, frames=frames, act="gelu", eps=1e-2)
    ops.group_norm(shape, gx.data_ptr(), 0, 0, y.data_ptr(), stats=stats.data_ptr(), stream=stream())
    ops.group_norm_grad(shape, gx.data_ptr(), 0, 0, stats.data_ptr(), gdy.data_ptr(), dx.data_ptr(), stream=stream())

    def loss(x):
        a = x.reshape(frames, rows // frames, groups, -1)
        m = a.mean((1, 3), keepdim=True)
        v = (a - m) / torch.sqrt((a - m).square().mean((1, 3), keepdim=True) + 1e-2)
        return (torch.nn.functional.gelu(v).reshape(rows, ch) * dy.double()).sum()

    for r, c in ((0, 0), (7, 11), (20, 5), (39, 3)):
        step = torch.zeros(rows, ch, dtype=torch.float64)
        step[r, c] = h
        slope = (loss(x.double() + step) - loss(x.double() - step)) / (2 * h)
        # second order: h^2 times third derivatives of up to about 10^3; fp32: 1e-5 of sums below 10
        assert abs(float(dx[r, c]) - float(slope)) < 1e-4 + 1e-4 * abs(float(slope))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 2, 3])
@pytest.mark.parametrize("ch,groups", [(32, 16), (96, 16), (35, 5), (64, 1), (8, 8), (9, 3), (7, 7)])
def test_checkpoints_of_a_few_rows(ops, dp, dtype, rows, ch, groups):
    """Frames named by starts, whose parts begin at any channel: reads of the checkpoint end with it."""
    norm_case(ops, dp, dtype, "silu", rows, ch, groups, lengths=[rows], kept=True, eps=1e-3)
    norm_case(ops, dp, dtype, "silu", rows, ch, groups, frames=1, kept=True, eps=1e-3)


@pytest.mark.parametrize("rows,ch,groups,frames", [(3000, 235, 47, 5), (2000, 1001, 7, 1), (900, 5005, 5, 2),
                                                   (700, 4100, 4100, 1), (260, 2310, 11, 260), (300, 9001, 1, 3),
                                                   (5000, 6, 2, 1), (1200, 12, 12, 40)])
def test_groups_across_vectors_and_parts(ops, dp, rows, ch, groups, frames):
    """Groups that no vector of 16 bytes divides, that go over several parts of the columns or are one
    channel each."""
    for k, dtype in enumerate(TYPES):
        norm_case(ops, dp, dtype, ("silu", "none", "gelu")[k], rows, ch, groups, frames)
        norm_case(ops, dp, dtype, ("gelu", "tanh", "none")[k], rows, ch, groups, frames, kept=True, eps=1e-3)


@pytest.mark.parametrize("rows,ch,groups,frames", [(70000, 1024, 32, 1), (70000, 1030, 103, 4), (70000, 1024, 16, 70000),
                                                   (70016, 1024, 64, 547)])
def test_outputs_past_the_caches(ops, dp, rows, ch, groups, frames):
    """Outputs of over 192 MB, which are stored in another way, in each form."""
    norm_case(ops, dp, "f32", "silu", rows, ch, groups, frames, at="cuda")


@pytest.mark.parametrize("frames", [1, "rows"])
def test_past_32_bits(ops, dp, frames):
    """More than 2^32 values: y, dx and the sums of the last rows, whose places pass 32 bits."""
    rows, ch, groups = 2 ** 21 + 32, 2080, 65
    x = torch.empty(rows, ch, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    for a in range(0, rows, 2 ** 18):
        x[a:a + 2 ** 18] = torch.randn(min(2 ** 18, rows - a), ch, generator=gen, device="cuda", dtype=torch.float32)
    n = rows if frames == "rows" else 1
    y, stats = torch.empty_like(x), torch.empty(n, groups, 2, device="cuda")
    shape = dp.ops.NormShape(rows, ch, groups, frames=n, dtype="bf16")
    ops.group_norm(shape, x.data_ptr(), 0, 0, y.data_ptr(), stats=stats.data_ptr(), stream=stream())
    dx, dgamma, dbeta = torch.empty_like(x), *(torch.empty(ch, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ops.group_norm_grad(shape, x.data_ptr(), 0, 0, stats.data_ptr(), y.data_ptr(), dx.data_ptr(), dgamma.data_ptr(),
                        dbeta.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    for part in (slice(0, 8), slice(rows - 8, rows)):
        a = x[part].double().reshape(8, groups, -1)
        if n == 1:
            # mean 0 and deviation 1 of 6.7e7 values each: off by 5 / sqrt of that, and its square root of two
            assert float(stats[0, :, 0].abs().max()) < 7e-4 and float((stats[0, :, 1] - 1).abs().max()) < 7e-4
            m, r = (stats[0, :, k].double()[:, None] for k in (0, 1))
        else:
            m = a.mean(2, keepdim=True)
            r = ((a - m).square().mean(2, keepdim=True) + 1e-5) ** -0.5
        want = ((a - m) * r).reshape(8, ch)
        got = y[part].double()
        assert bool(((got - want).abs() <= (2.0 ** -8 + 1e-5) * want.abs() + 1e-5).all())
        # dy = y = v (rounded): w = v, so dx = r (v - mean v - v mean v^2), small, as mean v^2 is nearly 1
        v, w = want.reshape(8, groups, -1), got.reshape(8, groups, -1)
        s1, s2 = (0.0, 1.0) if n == 1 else (w.mean(2, keepdim=True), (w * v).mean(2, keepdim=True))
        dxw = (r * (w - s1 - v * s2)).reshape(8, ch)
        # (n = 1: the means of w and w v to 1e-3, as above; both: rounded to bf16, terms of up to 5 in fp32)
        assert bool(((dx[part].double() - dxw).abs() <= 2.0 ** -8 * dxw.abs() + (1e-2 if n == 1 else 2e-5)).all())
    # dgamma = sum of y v, about the number of rows; dbeta = sum of y, a sum of 2^21 roundings and signs
    assert bool(((dgamma.double() / rows - 1).abs() < 2.0 ** -7).all())
    assert bool((dbeta.double().abs() < 6 * math.sqrt(rows)).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ch,groups", [(128, 32), (90, 18)])
def test_many_short_frames(ops, dp, dtype, ch, groups):
    """Thousands of frames of none to three rows (small molecules of a batch)."""
    lengths = [(7 * k) % 4 for k in range(3000)]
    norm_case(ops, dp, dtype, "silu", sum(lengths) + 5, ch, groups, lengths=lengths, first=2)


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("dtype,ch,groups", [("f32", 564, 4), ("bf16", 1064, 8), ("f16", 1100, 4), ("bf16", 2080, 16),
                                             ("f16", 2600, 4), ("f32", 2100, 3)])
def test_slices_of_uneven_widths(ops, dp, dtype, ch, groups, kept):
    """Rows that are cut into parts of columns, groups that go on beyond them."""
    norm_case(ops, dp, dtype, "silu", 4100, ch, groups, kept=kept)


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,ch,groups", [(37, 27, 3), (700, 90, 6), (300, 123, 3), (65, 235, 5), (130, 1010, 10),
                                            (40, 2500, 4), (33, 1476, 41), (9, 3999, 31), (21, 45, 5), (50, 4090, 409), (1000, 12, 2), (259, 30, 2),
                                            (300, 16, 4), (70, 3, 3)])
def test_rows_of_odd_groups(ops, dp, dtype, rows, ch, groups, kept):
    """Each row by itself, groups that end inside a thread's channels: of so many channels or more, and of fewer."""
    norm_case(ops, dp, dtype, "gelu", rows, ch, groups, frames=rows, kept=kept)


@pytest.mark.parametrize("shift", [30.0, 3000.0])
def test_rows_of_odd_groups_far_from_zero(ops, dp, shift):
    norm_case(ops, dp, "f32", "none", 64, 245, 7, frames=64, shift=shift)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ch,groups", [(4095, 1365), (4096, 4096), (2049, 2049), (62, 31), (64, 4), (61, 1), (33, 11)])
def test_rows_of_many_and_of_few_groups(ops, dp, dtype, ch, groups):
    """As many entries as a row may have in LDS, and rows of a few lanes."""
    norm_case(ops, dp, dtype, "silu", 90, ch, groups, frames=90)
