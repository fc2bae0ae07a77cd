"""Group norm of ragged frames of which one has nearly all rows, or most are empty: the work is cut by the mean length,
and the results are those of any frames."""
import pytest

from test_gpu_ops_norm import norm_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(dp):
    return dp.ops.Operators()


@pytest.mark.parametrize("dtype,kept", [("f32", False), ("bf16", True)])
@pytest.mark.parametrize("ch,groups", [(256, 32), (70, 7), (4200, 2)])
@pytest.mark.parametrize("lengths", [[1] * 60 + [6000] + [1] * 20, [0] * 900 + [5000, 3] + [0] * 98,
                                     [2] * 70 + [2000] + [0, 9] * 30])
def test_one_long_frame(ops, dp, dtype, kept, ch, groups, lengths):
    norm_case(ops, dp, dtype, "silu", sum(lengths) + 5, ch, groups, lengths=lengths, first=2, kept=kept, eps=1e-3)
