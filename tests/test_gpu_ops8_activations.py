"""The activations of the group norm and of the 8-bit products in 16 bits, and their derivatives, relative to
themselves, from small arguments to ones where the exponentials vanish.

The norm's argument is beta where gamma is zero; a row by itself has dbeta = dy act'(beta). The products' is one weight
times one input. gelu's Phi(-|g|) is allowed 2.5e-7, or 2^-15 of itself where that is less, and all of them the
roundings of test_gpu_ops_activations.py."""
import math

import pytest
import torch

from ops_reference import HALF_ULP, TINY, TORCH
from test_gpu_ops import stream
from test_gpu_ops_activations import NORMAL, exact

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(dp):
    return dp.ops.Operators()


def bounds(act, v, dtype):
    """((value, bound) of act, (value, bound) of act') in the type, v in 64 bits."""
    (a, ba), (da, bda) = exact(act, v)
    if act == "gelu":
        tail = torch.minimum(torch.tensor(2.5e-7, dtype=torch.float64), 2.0 ** -15 * 0.5 * torch.erfc(v.abs() / math.sqrt(2)))
        ba, bda = ba + v.abs() * tail, bda + tail
    return tuple((w, b + HALF_ULP[dtype] * (w.abs() + b) + TINY[dtype] + NORMAL * (1 + v.abs())) for w, b in ((a, ba), (da, bda)))


def check(what, v, got, want):
    over = (got.double().cpu() - want[0]).abs() - want[1]
    k = int(over.argmax())
    assert over[k] <= 0, (what, float(v[k]), float(got[k]), float(want[0][k]), float(want[1][k]))


def values(dtype):
    v = 10.0 ** torch.linspace(-6, 1.1, 1003, dtype=torch.float64)
    v[::2] *= -1
    return torch.cat([v, -torch.linspace(3, 12, 509, dtype=torch.float64)]).to(TORCH[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("act", ["tanh", "silu", "gelu"])
def test_norm(ops, dp, act, dtype):
    v = values(dtype)
    n = len(v)
    x, dy, gamma, beta = torch.randn(1, n).to(v.dtype).cuda(), torch.ones_like(v).cuda(), torch.zeros_like(v).cuda(), v.cuda()
    y, dbeta, stats = torch.empty_like(x), torch.empty_like(beta), torch.empty(1, 2, device="cuda")
    shape = dp.ops.NormShape(1, n, 1, dtype=dtype, act=act)
    ops.group_norm(shape, x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), y.data_ptr(), stats=stats.data_ptr(),
                   stream=stream())
    ops.group_norm_grad(shape, x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), stats.data_ptr(), dy.data_ptr(),
                        d_dbeta=dbeta.data_ptr(), stream=stream())
    a, da = bounds(act, v.double(), dtype)
    check("y", v, y[0], a)
    check("dbeta", v, dbeta, da)


@pytest.mark.parametrize("rows", [1, 20, 200])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("act", ["tanh", "silu", "gelu"])
def test_products(ops, dp, act, dtype, rows):
    """One input of 1 (127 / 127) and weights of 127 with scales v / 127: g is v to three roundings of 2^-24."""
    v = values(dtype)
    n = len(v)
    x = torch.ones(rows, 1, dtype=v.dtype, device="cuda")
    w = torch.zeros(n, 16, dtype=torch.int8, device="cuda")
    w[:, 0] = 127
    scale = (v.double() / 127).float().cuda()
    ones = torch.full((n,), 1 / 127, device="cuda")
    y = torch.empty(rows, n, dtype=v.dtype, device="cuda")
    shape = dp.ops.Linear8Shape(rows, 1, n, dtype=dtype, act=act)
    a = bounds(act, v.double(), dtype)[0]
    # (g's roundings, and those of the gate's factor: five of 2^-24 of values whose slope relative to them is at most
    # that of gelu, 1 + v^2)
    a = a[0], a[1] + 5 * 2.0 ** -24 * (2 + v.double() ** 2) * a[0].abs()
    for up in (False, True):
        more = dict(d_up=w.data_ptr(), d_up_scale=ones.data_ptr()) if up else {}
        ops.linear8(shape, x.data_ptr(), w.data_ptr(), scale.data_ptr(), y.data_ptr(), **more, stream=stream())
        check((rows, up), v, y[0], a)
        assert bool((y == y[0]).all())
