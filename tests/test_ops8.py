"""The 8-bit operators and the group norm where there is no GPU: refusals (arguments are looked at before
the device), and the 64-bit reference of the GPU tests against autograd, plain fp32 and its own definitions."""
import ctypes as C

import pytest
import torch

import ops8_reference as ref8
import ops_reference as ref


@pytest.fixture()
def handle(dp):
    """A handle of the library as the C caller gets it (kept where there is no GPU), and its calls."""
    L, h = dp.lib(), C.c_void_p()
    L.dp_ops_create(0, C.byref(h))
    assert h

    def refused(rc, text):
        assert rc == -1, rc  # DP_ERR_ARG
        assert text in L.dp_ops_last_error(h).decode()
    yield L, h, refused
    L.dp_ops_destroy(h)


A, B = 1 << 12, 1 << 13  # addresses that no call looks at


def test_keep8_refusals(dp, handle):
    L, h, refused = handle
    for args, text in (((7, 4, 32, A, 0, B), "unknown type"), ((0, -1, 32, A, 0, B), "rows"),
                       ((0, 2 ** 30 + 1, 32, A, 0, B), "rows"), ((0, 4, 0, A, 0, B), "cols"),
                       ((0, 4, 2 ** 20 + 1, A, 0, B), "cols"), ((0, 4, 32, A, 31, B), "ld_x"),
                       ((0, 4, 32, A, 2 ** 22 + 1, B), "ld_x"), ((0, 4, 32, A, 0, B + 8), "16-byte"),
                       ((0, 4, 32, None, 0, B), "null"), ((0, 4, 32, A, 0, None), "null")):
        refused(L.dp_keep8(h, *args, None), text)
        t, n, c, x, ld, k = args
        refused(L.dp_restore8(h, t, n, c, k, x, ld, None), text)
    assert L.dp_keep8(h, 0, 0, 32, None, 0, None, None) == 0
    assert L.dp_restore8(h, 0, 0, 32, None, None, 0, None) == 0
    assert L.dp_keep8(None, 0, 1, 32, A, 0, B, None) != 0


def test_keep8_bytes(dp):
    k = dp.ops.keep8_bytes
    assert k(1, 1) == 33 and k(3, 32) == 99 and k(3, 33) == 3 * 66 and k(0, 5) == 0
    assert k(2 ** 30, 2 ** 20) == 2 ** 30 * (2 ** 20 + 2 ** 15)
    assert k(-1, 5) == k(5, 0) == k(5, 2 ** 20 + 1) == k(2 ** 30 + 1, 5) == k(2 ** 64 + 1, 5) == k(1, 2 ** 32 + 1) == 0


def test_weights8_refusals(dp, handle):
    L, h, refused = handle
    for args, text in (((3, 64, 8, A, 0, A, 0, A), "unknown type"), ((0, 0, 8, A, 0, A, 0, A), "d_in"),
                       ((0, 2 ** 17 + 1, 8, A, 0, A, 0, A), "d_in"), ((0, 64, 0, A, 0, A, 0, A), "d_out"),
                       ((0, 64, 8, A, 7, A, 0, A), "ld_w"), ((0, 60, 8, A, 0, A, 60, A), "multiple of 16"),
                       ((0, 60, 8, A, 0, A, 48, A), "multiple of 16"), ((0, 64, 8, A, 0, A + 4, 0, A), "aligned"),
                       ((0, 64, 8, None, 0, A, 0, A), "null"), ((0, 64, 8, A, 0, A, 0, None), "null")):
        refused(L.dp_weights8(h, *args, None), text)


def test_linear8_refusals(dp, handle):
    L, h, refused = handle
    S = dp.ops.Linear8Shape

    def call(shape, x=A, w=A, ws=A, up=None, us=None, y=A):
        return L.dp_linear8(h, C.byref(shape.c), x, w, ws, up, us, y, None)

    for shape, text in ((S(4, 64, 8, dtype=9), "unknown type"), (S(4, 64, 8, act=4), "activation"),
                        (S(-1, 64, 8), "rows"), (S(2 ** 64 + 4, 64, 8), "rows"), (S(4, 0, 8), "d_in"),
                        (S(4, 2 ** 17 + 1, 8), "d_in"), (S(4, 2 ** 32 + 64, 8), "d_in"), (S(4, 64, 0), "d_out"),
                        (S(4, 64, 8, ld_x=63), "ld_x"), (S(4, 64, 8, ld_y=7), "ld_y"),
                        (S(4, 65, 8, ld_w=72), "multiple of 16"), (S(4, 65, 8, ld_w=64), "multiple of 16")):
        refused(call(shape), text)
    ok = S(4, 64, 8)
    for kw in ({"x": None}, {"w": None}, {"ws": None}, {"y": None}):
        refused(call(ok, **kw), "null")
    refused(call(ok, up=A), "both")
    refused(call(ok, us=A), "both")
    refused(call(ok, w=A + 8), "aligned")
    refused(call(ok, up=A + 8, us=A), "aligned")
    assert L.dp_linear8(h, None, A, A, A, None, None, A, None) != 0
    assert call(S(0, 64, 8), None, None, None, None, None, None) == 0


def test_backward8_refusals(dp, handle):
    L, h, refused = handle
    S = dp.ops.GatedShape

    def call(shape, kept=A, wg=A, wu=A, wd=A, dy=A, dx=A, dwg=None, dwu=None, dwd=None):
        return L.dp_gated_backward8(h, C.byref(shape.c), kept, wg, wu, wd, dy, dx, dwg, dwu, dwd, None)

    refused(call(S(4, 8, 8, 8, act="none")), "activation")  # (of the norm and the 8-bit products)
    refused(call(S(4, 0, 8, 8)), "d_in")
    ok = S(4, 8, 8, 8)
    refused(call(ok, dwg=A), "both")
    if not torch.cuda.is_available():  # (past the first checks these need the device)
        return
    refused(call(ok, kept=None), "null")
    refused(call(ok, kept=A + 8), "16-byte")
    refused(call(ok, dy=None), "null")


def test_norm_refusals(dp, handle):
    L, h, refused = handle
    S = dp.ops.NormShape

    def fwd(shape, x=A, starts=None, y=A, stats=None):
        return L.dp_group_norm(h, C.byref(shape.c), x, starts, None, None, y, stats, None)

    def grad(shape, x=A, kept=None, stats=A, dy=A, dx=A):
        return L.dp_group_norm_grad(h, C.byref(shape.c), x, kept, None, None, None, stats, dy, dx, None, None, None)

    for shape, text in ((S(8, 32, 4, dtype=5), "unknown type"), (S(8, 32, 4, act=7), "activation"),
                        (S(-1, 32, 4), "rows"), (S(8, 0, 4), "channels"), (S(8, 32, 0), "groups"),
                        (S(8, 32, 5), "groups"), (S(8, 32, 64), "groups"), (S(8, 32, 4, frames=0), "frames"),
                        (S(8, 32, 4, frames=3), "starts"), (S(8, 32, 4, eps=-1e-5), "eps"),
                        (S(8, 32, 4, eps=float("nan")), "eps"), (S(8, 32, 4, ld_x=31), "ld_x"),
                        (S(8, 32, 4, ld_y=31), "ld_y"), (S(8, 2 ** 32 + 32, 4), "channels"),
                        (S(8, 32, 4, frames=2 ** 32 + 1), "channels"), (S(8, 32, 4, ld_x=2 ** 64), "rows")):
        refused(fwd(shape), text)
        refused(grad(shape), text)
    ok = S(8, 32, 4, frames=2)
    refused(fwd(ok, x=None), "null")
    refused(fwd(ok, y=None), "null")
    refused(fwd(ok, stats=A + 4), "8-byte")
    refused(grad(ok, kept=A), "not both")
    refused(grad(ok, x=None, kept=A + 8), "16-byte")
    refused(grad(ok, stats=A + 4), "8-byte")
    assert fwd(S(0, 32, 4), None, None, None) == 0


@pytest.mark.parametrize("call,args", [("keep8", (16, 16, 4, 5)), ("restore8", (16, 16, 4, 5)),
                                       ("weights8", (16, 16, 16, 4, 5))])
def test_sizes_beyond_a_c_integer(dp, call, args):
    """They reach the library as -1, which it refuses."""
    from test_ops_sizes import Recorded
    ops = object.__new__(dp.ops.Operators)
    ops._h, ops._lib, ops._error = 1, Recorded(), dp.DeepmdException
    at = 2
    try:
        getattr(ops, call)(*args)
        assert ops._lib.args[at] == 4
        for k in range(len(args) - 2, len(args)):
            wide = list(args)
            wide[k] += 2 ** 64 if call != "weights8" and k == len(args) - 2 else 2 ** 32
            getattr(ops, call)(*wide)
            assert ops._lib.args[at] == -1
        getattr(ops, call)(*args, "f32", 2 ** 64 + 8)
        assert ops._lib.args[at] == -1
    finally:
        ops._h = None


# ---- the reference itself ---------------------------------------------------------------------
def test_checkpoint_definition():
    x = torch.tensor([[1.0, -0.5, 127.5 / 64, 0.0, 1.0 / 128, 3.0 / 128]], dtype=torch.float64)
    q, field = ref8.fields(x)
    assert field.tolist() == [[127]]  # unit 2^-6
    assert q[0, :6].tolist() == [64, -32, 127, 0, 0, 2]  # ties to even, 127.5 held at 127
    assert ref8.restored(x)[0].tolist() == [1.0, -0.5, 127 / 64, 0.0, 0.0, 2 / 64]
    big = torch.tensor([[float(torch.finfo(torch.float32).max), 2.0 ** -149]], dtype=torch.float64)
    assert ref8.restored(big)[0].tolist() == [127 * 2.0 ** 121, 0.0]
    small = torch.tensor([[2.0 ** -127, 2.0 ** -140]], dtype=torch.float64)
    assert ref8.restored(small)[0].tolist() == [2.0 ** -127, 0.0]
    assert torch.isnan(ref8.restored(torch.tensor([[1.0, float("inf")]], dtype=torch.float64))).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_a_checkpoint_is_of_the_type(dtype):
    """What is restored is a number of the type, and off by at most a unit."""
    gen = torch.Generator().manual_seed(3)
    t = ref.TORCH[dtype]
    for size in (1.0, 2.0 ** -24, 2.0 ** -130, 3e4, 2.0 ** 120):
        x = (torch.randn(40, 70, generator=gen, dtype=torch.float64) * size).to(t)
        x = torch.where(torch.isfinite(x), x, 0).double()
        r = ref8.restored(x)
        assert torch.equal(r.to(t).double(), r)
        unit = torch.pow(torch.tensor(2.0, dtype=torch.float64), ref8.fields(x)[1].double() - 133)
        assert ((r - x).abs() <= unit.repeat_interleave(32, 1)[:, :70]).all()


def test_row_scales():
    x = torch.tensor([[127.0, 63.5, -1.0], [0, 0, 0], [2.0 ** -120, 0, 0], [float("nan"), 1, 2]], dtype=torch.float64)
    q, s = ref8.rows8(x)
    assert q.tolist() == [[127, 64, -1], [0, 0, 0], [0, 0, 0], [0, 0, 0]]  # 63.5 to the even one
    assert s[:3, 0].tolist() == [1, 0, 0] and torch.isnan(s[3, 0])


@pytest.mark.parametrize("act", ["none", "tanh", "silu", "gelu"])
def test_norm_gradients(act):
    """The formulas of the backward are the derivative of the forward's; bounds hold for plain fp32, and
    catch one without eps or with the sample variance."""
    gen = torch.Generator().manual_seed(4)
    n, ch, groups, frames = 24, 30, 3, [(0, 8), (8, 0), (8, 1), (9, 15)]

    def rand(*s):
        return torch.randn(*s, generator=gen, dtype=torch.float64).float().double()

    x, dy, gamma, beta = rand(n, ch) + 0.5, rand(n, ch), rand(ch), rand(ch)
    want = ref8.norm("f32", act, x, gamma, beta, frames, groups, 1e-3, dy)

    def plain(x, gamma, beta, eps=1e-3, less=0):
        ys = []
        for first, count in frames:
            if count:
                a = x[first:first + count].reshape(count, groups, -1)
                m = a.mean((0, 2), keepdim=True)
                var = ((a - m) ** 2).sum((0, 2), keepdim=True) / (count * ch / groups - less)
                v = ((a - m) / torch.sqrt(var + eps)).reshape(count, ch)
                ys.append(act64(gamma * v + beta))
        return torch.cat(ys)

    def act64(z):
        return ref8.act64(act, z)[0]

    leaves = [t.clone().requires_grad_() for t in (x, gamma, beta)]
    for k, t in zip(("dx", "dgamma", "dbeta"), torch.autograd.grad(plain(*leaves), leaves, dy)):
        assert torch.allclose(want[k][0], t, rtol=1e-10, atol=1e-11), k
    v, b = want["y"]
    f = [t.float() for t in (x, gamma, beta)]
    assert ((plain(*f).double() - v).abs() <= b).all()
    assert not ((plain(*f, eps=0.0).double() - v).abs() <= b).all()
    assert not ((plain(*f, less=1).double() - v).abs() <= b).all()
