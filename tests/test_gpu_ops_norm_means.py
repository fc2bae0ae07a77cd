"""Group norm of values whose mean is a thousand deviations, against 64 bits and against what it says of m and r itself:
what (x - m) r loses is the rounding of m alone."""
import pytest
import torch

import ops8_reference as ref8
from ops_reference import HALF_ULP, TINY, TORCH
from test_gpu_ops import stream

pytestmark = pytest.mark.gpu
E32 = 2.0 ** -24

# each row a frame by lanes, by parts of two groups and by channels; frames of a block, and in slices
FORMS = [(64, 64, 4, 64), (64, 60, 4, 64), (64, 60, 20, 64), (640, 64, 4, 10), (640, 60, 20, 10), (20000, 64, 4, 1),
         (20000, 60, 20, 1)]


@pytest.fixture(scope="module")
def ops(dp):
    return dp.ops.Operators()


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,ch,groups,frames", FORMS)
def test_large_means(ops, dp, dtype, kept, rows, ch, groups, frames):
    """y is (x - m) r, and dgamma (of one row's dy in all) dy v: a difference, a product and a rounding to the type of
    exact m and r. m passes at most 64 additions (32 of a thread's values, its joins, the lanes'), the squares as
    many."""
    gen = torch.Generator().manual_seed(rows + ch)
    host = (torch.randn(rows, ch, generator=gen, dtype=torch.float64) + 1000.0).to(TORCH[dtype])
    if dtype != "f32":  # (whose numbers are 4 or 1/2 apart there)
        host = (torch.randn(rows, ch, generator=gen, dtype=torch.float64) * (4096 if dtype == "bf16" else 64) + 16384.0).to(TORCH[dtype])
    x, dy = host.cuda(), torch.zeros(rows, ch, dtype=host.dtype, device="cuda")
    row = rows // 2
    dy[row] = 1.0
    y, dgamma, stats = torch.empty_like(x), torch.empty(ch, dtype=x.dtype, device="cuda"), torch.empty(frames, groups, 2, device="cuda")
    shape = dp.ops.NormShape(rows, ch, groups, frames=frames, dtype=dtype, eps=1e-5)
    ops.group_norm(shape, x.data_ptr(), 0, 0, y.data_ptr(), stats=stats.data_ptr(), stream=stream())
    buf, given = None, x.data_ptr()
    if kept:
        buf = torch.empty(dp.ops.keep8_bytes(rows, ch), dtype=torch.uint8, device="cuda")
        ops.keep8(x.data_ptr(), buf.data_ptr(), rows, ch, dtype, stream=stream())
        given = 0
    ops.group_norm_grad(shape, given, 0, 0, stats.data_ptr(), dy.data_ptr(), d_dgamma=dgamma.data_ptr(),
                        kept=buf.data_ptr() if kept else 0, stream=stream())
    torch.cuda.synchronize()
    m, r = (t.double().cpu() for t in stats.unbind(-1))

    def spread(t):
        return t.repeat_interleave(rows // frames, 0).repeat_interleave(ch // groups, 1)

    def close(got, want):
        # (and half the distance of the smallest numbers: f16's below 2^-14 are 2^-24 apart)
        bound = (4 * E32 + HALF_ULP[dtype]) * want.abs() + TINY[dtype]
        over = (got.double().cpu() - want).abs() - bound
        assert float(over.max()) <= 0, (dtype, float(over.max()))

    a = host.double()
    close(y, (a - spread(m)) * spread(r))
    at = ref8.restored(a) if kept else a
    close(dgamma, ((at - spread(m)) * spread(r))[row])
    a = a.reshape(frames, rows // frames, groups, -1)
    mean = a.mean((1, 3))
    var = (a - mean[:, None, :, None]).square().mean((1, 3))
    # A part's mean that is off by d_i adds 2 n_i (m_i - m) d_i + n_i d_i^2 to the sum of squared deviations, over all
    # parts at most n (2 d sigma + d^2) with the largest d (Cauchy and Schwarz: sum of n_i (m_i - m)^2 <= n sigma^2); r is
    # off by half of that relative to n sigma^2.
    d = 64 * E32 * mean.abs()
    assert bool(((m - mean).abs() <= d).all())
    d = d / (var + 1e-5).sqrt()
    assert bool(((r * (var + 1e-5).sqrt() - 1).abs() <= 64 * E32 + d + d * d).all())
