"""Group norm of a frame whose values are more than 32-bit integers count."""
import pytest
import torch

from test_gpu_ops import stream

pytestmark = pytest.mark.gpu


def test_a_long_frame_among_empty_ones(dp):
    """2^28 rows and more of 16 channels in one of 1,100 frames, so that a block has all of them: rows times channels of
    a vector pass 2^31. The channels' halves lie one apart, which is part of the variance."""
    rows, ch, frames, at = 2 ** 28 + 2 ** 22, 16, 1100, 700
    x = torch.empty(rows, ch, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    x[:, 8:] += 1.0
    starts = torch.zeros(frames + 1, dtype=torch.int32, device="cuda")
    starts[at + 1:] = rows - 1  # (the last row is in no frame)
    y = torch.full_like(x, 7.0)
    stats = torch.empty(frames, 1, 2, device="cuda")
    ops, shape = dp.ops.Operators(), dp.ops.NormShape(rows, ch, 1, frames=frames, dtype="bf16")
    ops.group_norm(shape, x.data_ptr(), 0, 0, y.data_ptr(), stats=stats.data_ptr(), starts=starts.data_ptr(),
                   stream=stream())
    total = square = 0.0
    for part in x[:rows - 1].split(2 ** 24):
        part = part.double()
        total, square = total + part.sum(), square + part.square().sum()
    number = (rows - 1) * ch
    mean = total / number
    var = square / number - mean ** 2  # (in 64 bits, of values of one: 1e-12)
    r = (var + 1e-5) ** -0.5
    # A thread has 2^21 rows, joined in fours: 2^19 roundings of the mean (below 1) by 2^-25, and three of the sum
    # of squares by 2^-24 of itself, of which r has half.
    m, r32 = (float(v) for v in stats[at, 0])
    assert abs(m - float(mean)) < 2.0 ** -6 and abs(r32 / float(r) - 1) < 1.5 * 2.0 ** -5
    for k in (0, 12345678, 2 ** 28 + 5, rows - 2):
        want = (x[k].double() - m) * r32
        assert bool(((y[k].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-6).all())
    assert bool((y[rows - 1] == 7.0).all()) and float(stats[:at].abs().max()) == 0
