"""Training steps of the gated block at sizes that run every tile of every product, whole and sliced,
against 64 bits within the bounds of ops_reference.py."""
import pytest
import torch

from ops_tiles import SIZES, variants
from test_gpu_ops import gated_case

pytestmark = pytest.mark.gpu

ACTS = ("silu", "tanh", "gelu")


@pytest.mark.parametrize("dtype,size,act", [(t, s, ACTS[k % 3]) for t in ("f32", "bf16", "f16")
                                            for k, s in enumerate(SIZES["f32" if t == "f32" else "16"])])
def test_tiles(dp, dtype, size, act):
    gated_case(dp.ops.Operators(), dp, dtype, act, *size, seed=sum(size))


def test_tiles_of_this_card(dp):
    """The sizes are chosen for 256 compute units."""
    assert torch.cuda.get_device_properties(0).multi_processor_count == 256
    assert variants(dp, "bf16", *SIZES["16"][0])
