"""The operators of trainable heads on the GPU at the limits of their arguments and values."""
import pytest
import torch

import ops_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(dp):
    return dp.ops.Operators()


def stream():
    return torch.cuda.current_stream().cuda_stream


def test_lookup_of_no_rows(ops):
    """A tensor without elements has no address: no rows are looked up from and into such ones."""
    nothing = torch.empty(0, 8, device="cuda")
    ids = torch.empty(0, dtype=torch.int32, device="cuda")
    table = torch.ones(5, 8, device="cuda")
    assert nothing.data_ptr() == 0 and ids.data_ptr() == 0
    ops.embed(ids.data_ptr(), table.data_ptr(), nothing.data_ptr(), 0, 5, 8, stream=stream())
    dt = torch.full((5, 8), 7.0, device="cuda")
    ops.embed_grad(ids.data_ptr(), nothing.data_ptr(), dt.data_ptr(), 0, 5, 8, stream=stream())
    torch.cuda.synchronize()
    assert not dt.any()


def test_refusals_without_rows(dp, ops):
    """The sizes are checked where there are no rows too, and a table's gradient needs its table."""
    for args in ((0, 0, 8), (0, 5, 0), (0, 2 ** 30 + 1, 8)):
        with pytest.raises(dp.DeepmdException):
            ops.embed(0, 0, 0, *args)
    with pytest.raises(dp.DeepmdException, match="null"):
        ops.embed_grad(0, 0, 0, 0, 5, 8)


# ---- values at the limits of the types -------------------------------------------------------
def block(dp, ops, dtype, act, x, wg, wu, wd, dy=None):
    """y, and with dy also dx, dwg, dwu and dwd, on the CPU in 64 bits."""
    t = ref.TORCH[dtype]
    x, wg, wu, wd = (m.to(t).cuda().contiguous() for m in (x, wg, wu, wd))
    shape = dp.ops.GatedShape(*x.shape, *wd.shape, dtype=dtype, act=act)
    saved = torch.empty(shape.saved_bytes(), dtype=torch.uint8, device="cuda")
    y = torch.full((x.shape[0], wd.shape[1]), 7.0, dtype=t, device="cuda")
    w = [m.data_ptr() for m in (wg, wu, wd)]
    ops.gated_forward(shape, x.data_ptr(), *w, y.data_ptr(), saved=saved.data_ptr(), stream=stream())
    out = [y]
    if dy is not None:
        dy = dy.to(t).cuda()
        out += [torch.full_like(m, 7.0) for m in (x, wg, wu, wd)]
        ops.gated_backward(shape, x.data_ptr(), *w, saved.data_ptr(), dy.data_ptr(), *(m.data_ptr() for m in out[1:]),
                           stream=stream())
    torch.cuda.synchronize()
    return [m.double().cpu() for m in out]


def host(dtype, seed, n, d, f, o):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(r, c, generator=gen, dtype=torch.float64) * s).to(ref.TORCH[dtype]).double()
            for r, c, s in ((n, d, 1.0), (d, f, d ** -0.5), (d, f, d ** -0.5), (f, o, f ** -0.5), (n, o, 1.0))]


# (rows: kernels of their own up to eight; outputs: up to four)
FORMS = [(5, 24, 40, 12), (70, 24, 40, 12), (70, 24, 40, 1), (700, 200, 96, 24)]


@pytest.mark.parametrize("n,d,f,o", FORMS)
@pytest.mark.parametrize("act", ["tanh", "silu", "gelu"])
@pytest.mark.parametrize("dtype,size", [("f32", 300.0), ("f32", 1e15), ("bf16", 300.0), ("bf16", 1e15), ("f16", 16.0)])
def test_saturated_gates(dp, ops, dtype, size, act, n, d, f, o):
    """Pre-activations past the range of the exponentials (e^89 is infinite in 32 bits): finite, and
    within the bounds."""
    x, wg, wu, wd, dy = host(dtype, 3, n, d, f, o)
    x = (x * size).to(ref.TORCH[dtype]).double()
    got = block(dp, ops, dtype, act, x, wg, wu, wd, dy)
    want = ref.gated(dtype, act, x, wg, wu, wd, dy)
    for g, k in zip(got, ("y", "dx", "dwg", "dwu", "dwd")):
        v, b = want[k]
        assert torch.isfinite(v).all() and torch.isfinite(g).all(), k
        assert ((g - v).abs() <= b).all(), k


@pytest.mark.parametrize("n,d,f,o", FORMS)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_row_out_of_range_spoils_itself(dp, ops, dtype, bad, n, d, f, o):
    """y and dx of the other rows keep their bits; the weights' gradients are the sums that hold it."""
    x, wg, wu, wd, dy = host(dtype, 4, n, d, f, o)
    clean = block(dp, ops, dtype, "silu", x, wg, wu, wd, dy)
    x[3, 7] = bad
    got = block(dp, ops, dtype, "silu", x, wg, wu, wd, dy)
    keep = torch.arange(n) != 3
    for k in (0, 1):
        assert torch.equal(got[k][keep], clean[k][keep])
        assert not torch.isfinite(got[k][3]).any()
    for k in (2, 3):
        assert not torch.isfinite(got[k][7]).any()


@pytest.mark.parametrize("n,o", [(3, 5), (20, 5), (20, 1)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_infinities_are_kept(dp, ops, dtype, n, o):
    """With one hidden column (the seven beside it are the kernels' padding) an infinite x gives
    infinite outputs with their signs, not NaN from a padding zero times it."""
    inf = float("inf")
    x = torch.ones(n, 2, dtype=torch.float64)
    x[1, 0], x[2, 0] = inf, -inf
    wg, wu = torch.tensor([[1.0], [0.5]]).double(), torch.tensor([[2.0], [1.0]]).double()
    wd = torch.tensor([[1.0, -1.0, 0.25, 3.0, -8.0]]).double()[:, :o]
    got = block(dp, ops, dtype, "tanh", x, wg, wu, wd)[0]
    h = torch.tanh(x @ wg) * (x @ wu)  # inf and (-1)(-inf)
    assert torch.equal(got[1:3], (h @ wd)[1:3]) and torch.isinf(got[1:3]).all()
    assert torch.isfinite(got[[0] + list(range(3, n))]).all()


@pytest.mark.parametrize("n", [8, 9])
def test_f16_range_of_h(dp, ops, n):
    """h past the f16 range is infinite where it is rounded to it; the forward of up to eight rows keeps it."""
    x = torch.full((n, 1), 300.0, dtype=torch.float64)
    one = torch.ones(1, 1, dtype=torch.float64)
    wd = torch.full((1, 5), 0.25, dtype=torch.float64)
    dy = torch.ones(n, 5, dtype=torch.float64)
    y, dx, _, _, dwd = block(dp, ops, "f16", "silu", x, one, one, wd, dy)
    kept = float(torch.tensor(22500.0).half())
    assert bool((y == (kept if n == 8 else float("inf"))).all())
    assert torch.isinf(dwd).all()  # (the backward rounds h for any number of rows)
    assert torch.isfinite(dx).all()


@pytest.mark.parametrize("n,d,f,o", FORMS)
def test_f16_small_gradients(dp, ops, n, d, f, o):
    """Gradients among the f16 subnormals are within the bounds, which allow each rounding to the type
    (the matrix cores take subnormals); scaled by a power of two, as a caller
    scales its loss, the same gradients keep their digits."""
    x, wg, wu, wd, dy = host("f16", 6, n, d, f, o)
    small = (dy * 2.0 ** -17).half().double()
    for g in (small, small * 2.0 ** 14):
        got = block(dp, ops, "f16", "silu", x, wg, wu, wd, g)
        want = ref.gated("f16", "silu", x, wg, wu, wd, g)
        for k, name in ((1, "dx"), (2, "dwg"), (3, "dwu"), (4, "dwd")):
            v, b = want[name]
            assert ((got[k] - v).abs() <= b).all(), name
    for k in (1, 2, 3, 4):  # (in the scaled ones: half of the elements at least to a hundredth)
        v = want[("dx", "dwg", "dwu", "dwd")[k - 1]][0]
        assert ((got[k] - v).abs() <= 0.01 * v.abs()).double().mean() > 0.5
    # below half the smallest subnormal dg and du are zero, and with them dx
    tiny = torch.full_like(dy, 2.0 ** -24)
    dx = block(dp, ops, "f16", "silu", x, wg, wu, wd * 2.0 ** -8, tiny)[1]
    assert not dx.any()


# ---- the table's gradient --------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,vocab,width,ld", [(499800, 2, 8, 70), (499800, 16, 8, 8), (300001, 4, 5, 11),
                                              (100000, 2, 130, 130), (20000, 3, 1000, 1000), (400000, 1, 1, 3)])
def test_few_ids_many_rows(ops, dtype, n, vocab, width, ld):
    """Hundreds of blocks' tables, many steps a thread, exactly: whole numbers whose sums stay small."""
    t, gen = ref.TORCH[dtype], torch.Generator().manual_seed(n)
    ids = torch.randint(-1, vocab + 1, (n,), generator=gen)
    dout = torch.randint(-1, 2, (n, ld), generator=gen)
    # every pair of rows of one id cancels but for the last ones: sums that 16 bits hold
    ids, dout = ids.repeat_interleave(2)[:n], dout.repeat_interleave(2, 0)[:n]
    dout[1::2] *= -1
    dout[-200:] = torch.randint(-1, 2, (200, ld), generator=gen)
    d_ids, d_dout = ids.int().cuda(), dout.to(t).cuda()
    dt = torch.full((vocab, width), 7.0, dtype=t, device="cuda")
    at = d_dout.data_ptr() + (ld - width) * d_dout.element_size()
    ops.embed_grad(d_ids.data_ptr(), at, dt.data_ptr(), n, vocab, width, dtype, ld_dout=ld, stream=stream())
    ok = (ids >= 0) & (ids < vocab)
    want = torch.zeros(vocab, width, dtype=torch.float64).index_add_(0, ids[ok], dout[ok, ld - width:].double())
    torch.cuda.synchronize()
    assert torch.equal(dt.double().cpu(), want) and want.abs().max() <= 256


def test_other_ids_order(ops):
    """In the sorted form the bits of one id's sum do not depend on where the rows of the others are."""
    gen = torch.Generator().manual_seed(5)
    n, vocab, width, v = 20000, 3000, 96, 1234
    ids = torch.randint(0, vocab, (n,), generator=gen)
    mine = torch.rand(n, generator=gen) < 0.3
    ids[mine] = v
    dout = torch.randn(n, width, generator=gen)

    def grad(ids, dout):
        d_ids, d_dout = ids.int().cuda(), dout.cuda()
        dt = torch.empty(vocab, width, device="cuda")
        ops.embed_grad(d_ids.data_ptr(), d_dout.data_ptr(), dt.data_ptr(), n, vocab, width, stream=stream())
        return dt[v].cpu()

    one = grad(ids, dout)
    # all rows elsewhere, those of v in their order
    place = torch.randperm(n, generator=gen)
    own = (ids == v).nonzero()[:, 0]
    slots, _ = place[own].sort()
    place[own] = slots
    ids2, dout2 = torch.empty_like(ids), torch.empty_like(dout)
    ids2[place], dout2[place] = ids, dout
    assert not torch.equal(ids, ids2)
    assert torch.equal(grad(ids2, dout2), one)
    # (the sums do depend on the order of its own rows: the comparison can fail)
    dout2[slots] = dout2[slots].flip(0)
    assert not torch.equal(grad(ids2, dout2), one)
