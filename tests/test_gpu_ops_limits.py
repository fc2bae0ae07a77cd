"""The operators of trainable heads on the GPU at the limits of their arguments and values."""
import pytest
import torch

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
