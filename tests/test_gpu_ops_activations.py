"""The gated block's activations and their derivatives on the GPU, relative to themselves, from
tiny pre-activations to ones where the exponentials vanish.

Every other factor is made one: x = (v, 1), w_gate has one 1 (g = v), w_up another (u = 1),
w_down and dy hold ones, so that y is act(v), and dx is (act'(v), act(v)), with each product exact in
32 bits. Allowed are 2^-20 of the terms that a value is the sum of (about eight roundings), the
rounding of the exponentials' argument (2^-24 of it, twice), and in 16 bits the two roundings to the type."""
import math

import pytest
import torch

from ops_reference import HALF_ULP, TINY, TORCH

pytestmark = pytest.mark.gpu

UNIT, NORMAL = 2.0 ** -20, 2.0 ** -126


def exact(act, v):
    """((value, bound) of act, (value, bound) of act'), v in 64 bits."""
    z = v.abs()
    if act == "tanh":
        a, da = torch.tanh(v), torch.cosh(v) ** -2
        return (a, UNIT * a.abs()), (da, (UNIT + 2 * z * 2.0 ** -22) * da)
    if act == "silu":
        p, off = torch.sigmoid(v), UNIT + z * 2.0 ** -22
        a, da = v * p, p * (1 + v * (1 - p))
        return (a, off * a.abs()), (da, off * p * (1 + z))
    p, off = 0.5 * torch.erfc(-v / math.sqrt(2)), UNIT + v * v * 2.0 ** -22
    w = torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    a, da = v * p, p + v * w
    return (a, off * a.abs()), (da, off * (p + z * w))


def values(n, dtype):
    if n == 8:
        v = torch.tensor([1e-6, -1e-5, 1e-4, -1e-3, 1e-2, -0.3, 0.62, -1.1], dtype=torch.float64)
    else:
        v = 10.0 ** torch.linspace(-6, 1.3, n, dtype=torch.float64)
        v[::2] *= -1
    return v.to(TORCH[dtype])


# (eight rows and more, and one output, have kernels of their own)
@pytest.mark.parametrize("n,o", [(8, 8), (1001, 8), (1001, 1)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("act", ["tanh", "silu", "gelu"])
def test_activation(dp, act, dtype, n, o):
    t, d, f = TORCH[dtype], 8, 8
    v = values(n, dtype)
    x = torch.zeros(n, d, dtype=t)
    x[:, 0], x[:, 1] = v, 1
    wg, wu, wd = torch.zeros(d, f, dtype=t), torch.zeros(d, f, dtype=t), torch.eye(f, o, dtype=t)
    wg[0, 0] = wu[1, 0] = 1
    x, wg, wu, wd = (m.cuda() for m in (x, wg, wu, wd))
    dy = torch.zeros(n, o, dtype=t, device="cuda")
    dy[:, 0] = 1
    y, dx = torch.empty_like(dy), torch.empty_like(x)
    shape = dp.ops.GatedShape(n, d, f, o, dtype=dtype, act=act)
    saved = torch.empty(shape.saved_bytes(), dtype=torch.uint8, device="cuda")
    ops, st = dp.ops.Operators(), torch.cuda.current_stream().cuda_stream
    w = [m.data_ptr() for m in (wg, wu, wd)]
    ops.gated_forward(shape, x.data_ptr(), *w, y.data_ptr(), saved=saved.data_ptr(), stream=st)
    ops.gated_backward(shape, x.data_ptr(), *w, saved.data_ptr(), dy.data_ptr(), dx.data_ptr(), stream=st)
    torch.cuda.synchronize()
    a, da = exact(act, v.double())
    twice = 2 * HALF_ULP[dtype] if dtype != "f32" else HALF_ULP[dtype]
    for what, got, (want, bound) in (("y", y[:, 0], a), ("dx/du", dx[:, 1], a), ("dx/dg", dx[:, 0], da)):
        got = got.double().cpu()
        bound = bound + twice * (want.abs() + bound) + 2 * TINY[dtype] + NORMAL * (1 + v.double().abs())
        over = (got - want).abs() - bound
        k = int(over.argmax())
        assert over[k] <= 0, (what, float(v[k]), float(got[k]), float(want[k]), float(bound[k]))
