"""A training step of a head (lookup, gated block forward and backward, table gradient) captured
into one HIP graph and replayed on new inputs, between eager calls."""
import pytest
import torch

pytestmark = pytest.mark.gpu


# rows and table: in one block of the sort, tiles with their own starts, with scanned ones; by tables in LDS
@pytest.mark.parametrize("n,vocab,width", [(3000, 500, 24), (20000, 300, 24), (140000, 9000, 8), (3000, 2, 8)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("o", [1, 8])
def test_step_in_a_graph(dp, dtype, o, n, vocab, width):
    t = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    f, gen = 40, torch.Generator(device="cuda").manual_seed(n)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").to(t)

    table, wg, wu, wd, dy = normal(vocab, width), normal(width, f), normal(width, f), normal(f, o), normal(n, o)
    ids = torch.empty(n, dtype=torch.int32, device="cuda")
    shape = dp.ops.GatedShape(n, width, f, o, dtype=dtype)
    saved = torch.empty(shape.saved_bytes(), dtype=torch.uint8, device="cuda")
    x, dx = torch.empty(n, width, dtype=t, device="cuda"), torch.empty(n, width, dtype=t, device="cuda")
    outs = [torch.empty_like(dy)] + [torch.empty_like(m) for m in (wg, wu, wd, table)]
    y, dwg, dwu, dwd, dtable = outs

    def step(ops, st):
        ops.embed(ids.data_ptr(), table.data_ptr(), x.data_ptr(), n, vocab, width, dtype, scale=0.5, stream=st)
        w = [m.data_ptr() for m in (wg, wu, wd)]
        ops.gated_forward(shape, x.data_ptr(), *w, y.data_ptr(), saved=saved.data_ptr(), stream=st)
        ops.gated_backward(shape, x.data_ptr(), *w, saved.data_ptr(), dy.data_ptr(), dx.data_ptr(), dwg.data_ptr(),
                           dwu.data_ptr(), dwd.data_ptr(), stream=st)
        ops.embed_grad(ids.data_ptr(), dx.data_ptr(), dtable.data_ptr(), n, vocab, width, dtype, scale=0.5, stream=st)

    inputs = [torch.randint(-1, vocab + 1, (n,), generator=gen, device="cuda").int() for _ in range(3)]
    eager, captured, st = dp.ops.Operators(), dp.ops.Operators(), torch.cuda.Stream()
    want = []
    for new in inputs:
        ids.copy_(new)
        step(eager, torch.cuda.current_stream().cuda_stream)
        want.append([m.clone() for m in outs])
    torch.cuda.synchronize()
    step(captured, st.cuda_stream)  # the workspace of this stream
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        step(captured, st.cuda_stream)
    for k in (1, 2, 0, 0, 1):
        ids.copy_(inputs[k])
        for m in outs:
            m.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, ref in zip(outs, want[k]):
            assert torch.equal(got, ref)
        step(eager, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        for got, ref in zip(outs, want[k]):
            assert torch.equal(got, ref)


def test_a_workspace_that_a_graph_holds_outlives_its_growth(dp):
    """A larger eager call on the captured stream gets a new workspace; the graph keeps its own."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    d, f, o = 30, 70, 12  # (odd rows: x and the weights are copied into the workspace, beside h)
    w = [torch.randn(*s, generator=gen, device="cuda") for s in ((d, f), (d, f), (f, o))]
    ops, st = dp.ops.Operators(), torch.cuda.Stream()

    def forward(x, y, stream):
        ops.gated_forward(dp.ops.GatedShape(len(x), d, f, o), x.data_ptr(), *(m.data_ptr() for m in w), y.data_ptr(),
                          stream=stream)

    x, big = (torch.randn(n, d, generator=gen, device="cuda") for n in (100, 20000))
    y, want, other = torch.empty(100, o, device="cuda"), torch.empty(100, o, device="cuda"), torch.empty(20000, o,
                                                                                                     device="cuda")
    torch.cuda.synchronize()
    forward(x, want, st.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        forward(x, y, st.cuda_stream)
    small = ops.device_bytes()
    for _ in range(3):
        forward(big, other, st.cuda_stream)
        torch.cuda.synchronize()
        assert ops.device_bytes() > small
        fill = torch.full((4 << 20,), float("nan"), device="cuda")  # (would take a freed workspace's place)
        y.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and bool(torch.isnan(fill).all())
