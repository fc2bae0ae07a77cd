"""The operators' front end where there is no GPU, and the 64-bit reference that the GPU tests
use: its gradients against autograd's, its bounds against a plain fp32 evaluation."""
import pytest
import torch

import ops_reference as ref


def test_no_gpu_is_an_error(dp):
    if torch.cuda.is_available():
        pytest.skip("a GPU is here")
    with pytest.raises(dp.DeepmdException, match="dp_ops_create"):
        dp.ops.Operators()


def test_saved_bytes(dp):
    S = dp.ops.GatedShape
    assert S(7, 3, 5, 2).saved_bytes() == 8 * 7 * 5
    assert S(0, 3, 5, 2).saved_bytes() == 0
    assert S(2 ** 30, 3, 2 ** 20, 2).saved_bytes() == 8 * 2 ** 50
    for bad in (S(-1, 3, 5, 2), S(7, 0, 5, 2), S(7, 3, 5, 2, dtype="int8"), S(7, 3, 5, 2, ld_hidden=4)):
        assert bad.saved_bytes() == 0


def inputs(dtype, n=9, d=12, f=20, o=5):
    gen = torch.Generator().manual_seed(1)
    mats = [torch.randn(s, generator=gen, dtype=torch.float64) * (s[0] ** -0.5 if k in (1, 2, 3) else 1.0)
            for k, s in enumerate(((n, d), (d, f), (d, f), (f, o), (n, o)))]
    return [m.to(ref.TORCH[dtype]).double() for m in mats]


@pytest.mark.parametrize("act", ["tanh", "silu", "gelu"])
def test_reference_gradients(act):
    """The formulas of the backward are the derivative of the forward's."""
    *leaves, dy = inputs("f32")
    want = ref.gated("f32", act, *leaves, dy)
    for t in leaves:
        t.requires_grad_()
    y = ref.gated("f32", act, *leaves)["y"][0]
    grads = torch.autograd.grad(y, leaves, dy)
    for k, g in zip(("dx", "dwg", "dwu", "dwd"), grads):
        assert torch.allclose(want[k][0], g, rtol=1e-12, atol=1e-12), k


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_bounds_hold_and_catch(dtype):
    """A plain evaluation in 32 bits, rounded where the kernels round, is within the bounds;
    one with a wrong activation, or a product short of one term, is not."""
    t = ref.TORCH[dtype]

    def short(kind, cut):
        x, wg, wu, wd, dy = (m.float() for m in inputs(dtype))
        k = x.shape[1] - cut
        g, u = x[:, :k] @ wg[:k], x @ wu
        a = torch.nn.functional.silu(g) if kind == "silu" else torch.tanh(g)
        return (((a * u).to(t).float()) @ wd).to(t).double()

    x, wg, wu, wd, _ = inputs(dtype)
    v, b = ref.gated(dtype, "silu", x, wg, wu, wd)["y"]
    assert ((short("silu", 0) - v).abs() <= b).all()
    assert not ((short("tanh", 0) - v).abs() <= b).all()
    assert not ((short("silu", 1) - v).abs() <= b).all()


def test_embed_reference():
    ids = torch.tensor([0, 2, -1, 3, 2, 7])
    table = torch.arange(8.0, dtype=torch.float64).reshape(4, 2)
    v, _ = ref.embed("f32", ids, table, 2.0)
    assert v.tolist() == [[0, 2], [8, 10], [0, 0], [12, 14], [8, 10], [0, 0]]
    g, _ = ref.embed_grad("f32", ids, torch.ones(6, 2, dtype=torch.float64), 4, 0.5)
    assert g.tolist() == [[0.5, 0.5], [0, 0], [1, 1], [0.5, 0.5]]
