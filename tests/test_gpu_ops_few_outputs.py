"""The gated block with up to four outputs in 16 bits: h meets no matrix core there, and y and dw_down come
from it unrounded, rounded once themselves."""
import pytest
import torch

import ops_reference as ref
from test_gpu_ops_limits import block, host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(dp):
    return dp.ops.Operators()


# (few rows have kernels of their own; the third gate is cut into slices; the last has one wave a row)
@pytest.mark.parametrize("n,d,f", [(5, 40, 200), (300, 40, 203), (9, 4096, 72), (33, 24, 2041)])
@pytest.mark.parametrize("o", [1, 3, 4])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_one_rounding(dp, ops, dtype, o, n, d, f):
    x, wg, wu, wd, dy = host(dtype, n + o, n, d, f, o)
    y, _, _, _, dwd = block(dp, ops, dtype, "silu", x, wg, wu, wd, dy)
    g, u = x @ wg, x @ wu
    bg, bu = ref.gamma(d) * (x.abs() @ wg.abs()), ref.gamma(d) * (x.abs() @ wu.abs())
    a, _ = ref.act64("silu", g)
    h = a * u
    bh = (ref.SLOPE * u.abs() * bg + a.abs() * bu + ref.SLOPE * bg * bu + ref.ACT * (1 + a.abs()) * u.abs())
    half, tiny = ref.HALF_ULP[dtype], ref.TINY[dtype]
    for got, v, m, k in ((y, h @ wd, (bh @ wd.abs(), (h.abs() + bh) @ wd.abs()), f),
                         (dwd, h.T @ dy, (bh.T @ dy.abs(), (h.abs() + bh).T @ dy.abs()), n)):
        b = m[0] + ref.gamma(k) * m[1]
        b = b + half * (v.abs() + b) + tiny
        assert ((got - v).abs() <= b).all(), float(((got - v).abs() - b).max())


@pytest.mark.parametrize("n", [8, 9, 300])
def test_range(dp, ops, n):
    """h beyond the f16 range: what is formed from it is finite."""
    x = torch.full((n, 1), 300.0, dtype=torch.float64)
    one = torch.ones(1, 1, dtype=torch.float64)
    y, _, _, _, dwd = block(dp, ops, "f16", "silu", x, one, one, one * 0.25, torch.full((n, 1), 2.0 ** -10).double())
    assert bool((y == float(torch.tensor(22500.0).half())).all())
    assert float(dwd) == float(torch.tensor(n * 90000 * 2.0 ** -10).half())
