"""Group norm at the ends of fp32's range and at lengths whose products leave 32-bit integers, in each of its
forms: rows by themselves, frames of a block, frames in slices."""
import math

import pytest
import torch

from test_gpu_ops import stream

pytestmark = pytest.mark.gpu

# rows, channels, groups, frames: as above, the last two in slices
FORMS = [(64, 64, 4, 64), (640, 64, 4, 10), (20000, 64, 4, 1), (20000, 65, 5, 1)]
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops(dp):
    return dp.ops.Operators()


def norm(ops, dp, x, groups, frames, eps, starts=0):
    """y and stats of x without gamma and beta."""
    dtype = next(k for k, t in TYPES.items() if t == x.dtype)
    y, stats = torch.zeros_like(x), torch.empty(frames, groups, 2, device="cuda")
    shape = dp.ops.NormShape(*x.shape, groups, frames=frames, dtype=dtype, eps=eps)
    ops.group_norm(shape, x.data_ptr(), 0, 0, y.data_ptr(), stats=stats.data_ptr(), starts=starts, stream=stream())
    torch.cuda.synchronize()
    return y, stats


@pytest.mark.parametrize("dtype,step", [("f32", 54), ("bf16", 58)])
@pytest.mark.parametrize("rows,ch,groups,frames", FORMS)
def test_means_whose_squares_leave_the_range(ops, dp, dtype, step, rows, ch, groups, frames):
    """2^65 and one step more: the mean's square passes 2^128, those of the deviations and their sums (in bf16 of a
    slice's rows) do not. The mean is off by 32 roundings of a batch's sum and one of each of at most 320 joins,
    2^-24 of it each: below 352 * 2^41 < 2^50, an eighth of the deviations (2^53 and more); y (one in magnitude) by that
    and by its rounding."""
    gen = torch.Generator().manual_seed(rows + ch)
    x = (2.0 ** 65 + 2.0 ** step * torch.randint(0, 2, (rows, ch), generator=gen).double()).to(TYPES[dtype])
    y, _ = norm(ops, dp, x.cuda(), groups, frames, 0.0)
    a = x.double().reshape(frames, rows // frames, groups, -1)
    m = a.mean((1, 3), keepdim=True)
    want = ((a - m) / (a - m).square().mean((1, 3), keepdim=True).sqrt()).reshape(rows, ch)
    assert bool(torch.isfinite(y).all())
    assert float((y.double().cpu() - want).abs().max()) < 0.25 * float(want.abs().max())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,ch,groups,frames", FORMS)
def test_deviations_whose_squares_leave_the_range(ops, dp, dtype, rows, ch, groups, frames):
    """Deviations of 10^20: their group is NaN, as with an infinity, and not act(beta); other groups are not."""
    gen = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, ch, generator=gen)
    x[:, ch // groups:2 * ch // groups] *= 1e20
    y, stats = norm(ops, dp, x.to(TYPES[dtype]).cuda(), groups, frames, 1e-5)
    bad = torch.zeros(ch, dtype=torch.bool)
    bad[ch // groups:2 * ch // groups] = True
    assert bool(torch.isnan(y[:, bad]).all()) and bool(torch.isfinite(y[:, ~bad]).all())
    assert bool(torch.isnan(stats[:, 1, 1]).all())


@pytest.mark.parametrize("rows,ch,groups,frames", FORMS)
def test_variances_below_the_normal_numbers(ops, dp, rows, ch, groups, frames):
    """Deviations of 2^-70 with eps 0: a variance below 2^-126 counts as zero, whose r is infinite, in each form; one of
    2^-122 does not."""
    gen = torch.Generator().manual_seed(rows)
    sign = torch.randint(0, 2, (rows, ch), generator=gen).float() * 2 - 1
    y, stats = norm(ops, dp, (sign * 2.0 ** -70).cuda(), groups, frames, 0.0)
    assert bool((stats[..., 1] == math.inf).all()) and not bool(torch.isfinite(y).any())
    y, stats = norm(ops, dp, (sign * 2.0 ** -61).cuda(), groups, frames, 0.0)
    assert bool(torch.isfinite(y).all()) and bool(torch.isfinite(stats).all())
    # (an eps of its own makes both ordinary)
    y, stats = norm(ops, dp, (sign * 2.0 ** -70).cuda(), groups, frames, 2.0 ** -100)
    assert bool((y.abs() < 2.0 ** -19).all()) and bool((stats[..., 1] == 2.0 ** 50).all())
