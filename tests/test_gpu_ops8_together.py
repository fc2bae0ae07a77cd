"""The operators around the gated block as they are used together: a layer's training step (norm of ragged cells,
block, both trained from 8-bit checkpoints) against 64 bits stage by stage, and the same layer served in 8 bits; the step and
the serving captured into HIP graphs, on several streams, and refusals inside a capture."""
import pytest
import torch

import ops8_reference as ref8
import ops_reference as ref
from test_gpu_ops import check

pytestmark = pytest.mark.gpu


class Layer:
    """x -> norm, silu -> gated block; cells of atoms as frames, the last rows padding."""

    def __init__(self, dp, dtype, lengths, d, groups, f, o, seed=0):
        self.dp, self.dtype, self.t = dp, dtype, ref.TORCH[dtype]
        self.lengths, self.n, self.d, self.groups, self.f, self.o = lengths, sum(lengths) + 3, d, groups, f, o
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.gen = gen

        def normal(*shape, size=1.0):
            return (torch.randn(*shape, generator=gen, device="cuda") * size).to(self.t)

        n = self.n
        self.x, self.dy = normal(n, d), normal(n, o)
        self.gamma, self.beta = normal(d), normal(d)
        self.w = [normal(d, f, size=d ** -0.5), normal(d, f, size=d ** -0.5), normal(f, o, size=f ** -0.5)]
        ends = torch.cumsum(torch.tensor([0] + lengths), 0)
        self.starts = ends.int().cuda()
        self.norm = dp.ops.NormShape(n, d, groups, frames=len(lengths), dtype=dtype, act="silu", eps=1e-3)
        self.block = dp.ops.GatedShape(n, d, f, o, dtype=dtype, act="gelu")
        self.out = {"h": torch.zeros(n, d, dtype=self.t, device="cuda"), "y": torch.empty_like(self.dy),
                    "stats": torch.empty(len(lengths), groups, 2, device="cuda"),
                    "dh": torch.empty(n, d, dtype=self.t, device="cuda"),
                    "dx": torch.zeros(n, d, dtype=self.t, device="cuda"), "dgamma": torch.empty_like(self.gamma),
                    "dbeta": torch.empty_like(self.beta), "dwg": torch.empty_like(self.w[0]),
                    "dwu": torch.empty_like(self.w[1]), "dwd": torch.empty_like(self.w[2])}
        self.kept_x, self.kept_h = (torch.empty(dp.ops.keep8_bytes(n, d), dtype=torch.uint8, device="cuda")
                                    for _ in range(2))

    def train(self, ops, st):
        p = {k: v.data_ptr() for k, v in self.out.items()}
        w = [m.data_ptr() for m in self.w]
        g, b, s = self.gamma.data_ptr(), self.beta.data_ptr(), self.starts.data_ptr()
        ops.group_norm(self.norm, self.x.data_ptr(), g, b, p["h"], stats=p["stats"], starts=s, stream=st)
        ops.keep8(self.x.data_ptr(), self.kept_x.data_ptr(), self.n, self.d, self.dtype, stream=st)
        ops.gated_forward(self.block, p["h"], *w, p["y"], stream=st)
        ops.keep8(p["h"], self.kept_h.data_ptr(), self.n, self.d, self.dtype, stream=st)
        ops.gated_backward8(self.block, self.kept_h.data_ptr(), *w, self.dy.data_ptr(), p["dh"], p["dwg"], p["dwu"],
                            p["dwd"], stream=st)
        ops.group_norm_grad(self.norm, 0, g, b, p["stats"], p["dh"], p["dx"], p["dgamma"], p["dbeta"],
                            kept=self.kept_x.data_ptr(), starts=s, stream=st)

    def pack(self, ops, st):
        """The block's weights in 8 bits, and what serving needs."""
        self.w8, self.scale = [], []
        for m in self.w:
            d, o = m.shape
            self.w8.append(torch.empty(o, (d + 15) // 16 * 16, dtype=torch.int8, device="cuda"))
            self.scale.append(torch.empty(o, device="cuda"))
            ops.weights8(m.data_ptr(), self.w8[-1].data_ptr(), self.scale[-1].data_ptr(), d, o, self.dtype, stream=st)
        self.gate8 = self.dp.ops.Linear8Shape(self.n, self.d, self.f, dtype=self.dtype, act="gelu")
        self.down8 = self.dp.ops.Linear8Shape(self.n, self.f, self.o, dtype=self.dtype)
        self.served = {"h": torch.zeros_like(self.out["h"]),
                       "a": torch.empty(self.n, self.f, dtype=self.t, device="cuda"), "y": torch.empty_like(self.dy)}

    def serve(self, ops, st):
        p = {k: v.data_ptr() for k, v in self.served.items()}
        w, s = [m.data_ptr() for m in self.w8], [m.data_ptr() for m in self.scale]
        ops.group_norm(self.norm, self.x.data_ptr(), self.gamma.data_ptr(), self.beta.data_ptr(), p["h"],
                       starts=self.starts.data_ptr(), stream=st)
        ops.linear8(self.gate8, p["h"], w[0], s[0], p["a"], d_up=w[1], d_up_scale=s[1], stream=st)
        ops.linear8(self.down8, p["a"], w[2], s[2], p["y"], stream=st)


SHAPES = [([40, 0, 7, 1, 60], 48, 6, 80, 24), ([200, 100], 70, 7, 96, 1), ([3], 100, 4, 200, 9)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lengths,d,groups,f,o", SHAPES)
def test_a_layer(dp, dtype, lengths, d, groups, f, o):
    """Each stage against 64 bits at the outputs of the stages before it."""
    ops, layer = dp.ops.Operators(), Layer(dp, dtype, lengths, d, groups, f, o)
    st = torch.cuda.current_stream().cuda_stream
    layer.train(ops, st)
    layer.pack(ops, st)
    layer.serve(ops, st)
    torch.cuda.synchronize()
    host = {k: v.cpu().double() for k, v in layer.out.items()}
    served = {k: v.cpu().double() for k, v in layer.served.items()}
    x, dy, gamma, beta = (v.cpu().double() for v in (layer.x, layer.dy, layer.gamma, layer.beta))
    w = [m.cpu().double() for m in layer.w]
    first, parts = 0, []
    for k in lengths:
        parts.append((first, k))
        first += k
    rows = slice(0, sum(lengths))  # (the others are padding)
    want = ref8.norm(dtype, "silu", x, gamma, beta, parts, groups, 1e-3, host["dh"], ref8.restored(x))
    for k in ("dgamma", "dbeta"):
        check(host[k], want[k], k)
    for k, got in (("y", host["h"]), ("dx", host["dx"]), ("y", served["h"])):
        check(got[rows], tuple(v[rows] for v in want[k]), k)
        assert bool((got[rows.stop:] == 0).all())
    check(host["y"], ref.gated(dtype, "gelu", host["h"], *w)["y"], "block")
    back = ref.gated(dtype, "gelu", ref8.restored(host["h"]), *w, dy)
    for k, key in (("dh", "dx"), ("dwg", "dwg"), ("dwu", "dwu"), ("dwd", "dwd")):
        check(host[k], back[key], k)
    q, s = zip(*(ref8.rows8(m.T.contiguous()) for m in w))
    a = ref8.linear8(dtype, "gelu", served["h"], q[0], s[0][:, 0], q[1], s[1][:, 0])
    check(served["a"], a, "gate8")
    check(served["y"], ref8.linear8(dtype, "none", served["a"], q[2], s[2][:, 0]), "down8")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lengths,d,groups,f,o", SHAPES + [([900, 50, 700], 264, 33, 520, 264)])
def test_in_a_graph(dp, dtype, lengths, d, groups, f, o):
    """Step and serving captured, and replayed on new inputs between eager calls: the same bits."""
    layer, eager, captured, st = Layer(dp, dtype, lengths, d, groups, f, o), dp.ops.Operators(), dp.ops.Operators(), \
        torch.cuda.Stream()
    layer.pack(eager, torch.cuda.current_stream().cuda_stream)

    def outputs():
        return [*layer.out.values(), *layer.served.values()]

    def step(ops, s):
        layer.train(ops, s)
        layer.serve(ops, s)

    inputs = [torch.randn(layer.n, d, generator=layer.gen, device="cuda").to(layer.t) for _ in range(3)]
    want = []
    for new in inputs:
        layer.x.copy_(new)
        step(eager, torch.cuda.current_stream().cuda_stream)
        want.append([m.clone() for m in outputs()])
    torch.cuda.synchronize()
    step(captured, st.cuda_stream)  # the workspace of this stream
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        step(captured, st.cuda_stream)
    for k in (1, 2, 0, 0, 1):
        layer.x.copy_(inputs[k])
        for name, m in [*layer.out.items(), *layer.served.items()]:
            m.fill_(0.0 if name in ("h", "dx") else 7.0)  # (padding of these two is left as it was)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(outputs(), want[k]):
            assert torch.equal(got, w)
        step(eager, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        for got, w in zip(outputs(), want[k]):
            assert torch.equal(got, w)


def test_two_streams(dp):
    """One handle on two streams at once, each with its own layer: as one after the other."""
    ops = dp.ops.Operators()
    layers = [Layer(dp, "bf16", [700, 300], 256, 16, 512, 64, seed=1), Layer(dp, "bf16", [5, 6, 900], 70, 7, 300, 3, seed=2)]
    streams = [torch.cuda.Stream() for _ in layers]
    want = []
    for layer in layers:
        layer.pack(ops, 0)
        layer.train(ops, 0)
        layer.serve(ops, 0)
        torch.cuda.synchronize()
        want.append([v.clone() for v in (*layer.out.values(), *layer.served.values())])
    torch.cuda.synchronize()
    for _ in range(5):
        for layer, st in zip(layers, streams):
            layer.train(ops, st.cuda_stream)
            layer.serve(ops, st.cuda_stream)
    torch.cuda.synchronize()
    for layer, w in zip(layers, want):
        for got, v in zip((*layer.out.values(), *layer.served.values()), w):
            assert torch.equal(got, v)


def test_a_capture_without_a_workspace_is_refused(dp):
    """The calls that need one say so, the capture goes on without them, and the handle serves later calls."""
    ops, st = dp.ops.Operators(), torch.cuda.Stream()
    layer = Layer(dp, "f32", [3000, 3000], 64, 8, 96, 8)
    layer.pack(dp.ops.Operators(), 0)
    torch.cuda.synchronize()
    p = {k: v.data_ptr() for k, v in layer.out.items()}
    one = dp.ops.NormShape(layer.n, 64, 8, dtype="f32")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        s = st.cuda_stream
        with pytest.raises(dp.DeepmdException, match="cannot grow"):
            ops.gated_backward8(layer.block, layer.kept_h.data_ptr(), *(m.data_ptr() for m in layer.w),
                                layer.dy.data_ptr(), p["dh"], stream=s)
        with pytest.raises(dp.DeepmdException, match="cannot grow"):
            ops.linear8(layer.gate8, p["h"], layer.w8[0].data_ptr(), layer.scale[0].data_ptr(),
                        layer.served["a"].data_ptr(), stream=s)
        with pytest.raises(dp.DeepmdException, match="cannot grow"):
            ops.group_norm_grad(one, layer.x.data_ptr(), 0, 0, p["stats"], p["h"], p["dx"], p["dgamma"], stream=s)
        ops.keep8(layer.x.data_ptr(), layer.kept_x.data_ptr(), layer.n, 64, stream=s)  # (needs none)
    graph.replay()
    layer.train(ops, st.cuda_stream)
    torch.cuda.synchronize()
    again = dp.ops.Operators()
    first = {k: v.clone() for k, v in layer.out.items()}
    layer.train(again, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(first[k], layer.out[k]) for k in first)
