"""The gated block's gradients from a checkpoint at sizes that run every tile of its own products, whole and sliced,
against 64 bits within the bounds of ops_reference.py."""
import pytest
import torch

from ops8_tiles import HEADS, SIZES
from test_gpu_ops8 import backward8_case

pytestmark = pytest.mark.gpu
ACTS = ("silu", "tanh", "gelu")


@pytest.fixture(scope="module")
def ops(dp):
    return dp.ops.Operators()


@pytest.mark.parametrize("dtype,size,act", [(t, s, ACTS[k % 3]) for t in ("f32", "bf16", "f16")
                                            for k, s in enumerate(HEADS + SIZES["f32" if t == "f32" else "16"])])
def test_tiles(ops, dp, dtype, size, act):
    backward8_case(ops, dp, dtype, act, *size)


@pytest.mark.parametrize("which", [("dx",), ("dwg", "dwu"), ("dwd",)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size,pad,skip", [((192, 1600, 240, 240), 0, 0), ((193, 1601, 241, 2), 3, 1),
                                           ((577, 77, 1783, 3943), 8, 8)])
def test_some_of_a_sliced_call(ops, dp, dtype, size, pad, skip, which):
    """Some of the outputs, rows with gaps, where gate and dh are cut."""
    backward8_case(ops, dp, dtype, "silu", *size, pad=pad, skip=skip, which=which)


@pytest.mark.parametrize("size", [HEADS[0], HEADS[1], (577, 77, 1783, 3943)])
def test_sliced_calls_repeat(ops, dp, size):
    first = backward8_case(ops, dp, "bf16", "gelu", *size)
    again = backward8_case(ops, dp, "bf16", "gelu", *size)
    assert all(torch.equal(first[k], again[k]) for k in first)
