"""The sizes of ops8_tiles.py reach every tile that the library takes for a product of the gated block's gradients from
a checkpoint on 256 compute units, whole and sliced (what it takes is asked of it for shapes drawn over the range)."""
import math
import random

import pytest

from ops8_tiles import HEADS, SIZES, variants


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_every_tile_is_run(dp, dtype):
    rng = random.Random(dtype)

    def size(lo, hi, whole):
        v = round(math.exp(rng.uniform(math.log(lo), math.log(hi))))
        return max(8, v // 8 * 8) if whole else v | 1

    taken = set()
    for _ in range(30000):
        whole = rng.random() < 0.4
        taken |= variants(dp, dtype, size(1, 100000, whole), size(16, 4096, whole), size(16, 8192, whole),
                          rng.choice([1, 2, 3, 4]) if rng.random() < 0.4 and not whole else size(5, 4096, whole))
    run = set().union(*(variants(dp, dtype, *s) for s in SIZES["f32" if dtype == "f32" else "16"]))
    assert len(taken) > 50 and taken <= run
    # dh in several sums beside a whole and a sliced gate, and the gate of few outputs that keeps g and u
    assert {(a, b) for a in (False, True) for b in (False, True)} == {(v[1], v[3]) for v in run if v[2] == "dh"}
    assert any(v[0] == "gate" for v in run)


def test_heads_are_sliced(dp):
    """A head on a few cells' descriptors: few rows, a long sum."""
    for s in HEADS:
        plan = dp.ops.GatedShape(*s, dtype="bf16").plan8()
        assert plan["gate" if s[3] <= 4 else "gate_back"][2] > 1, s


def test_plan(dp):
    S = dp.ops.GatedShape
    assert set(S(9, 16, 16, 5).plan8()) == {"gate_back", "dh", "dx", "dw", "dw_down"}
    assert set(S(9, 16, 16, 4).plan8()) == {"gate_outs", "dx", "dw"}
    assert set(S(9, 16, 16, 1).plan8()) == {"gate_one", "dx", "dw"}
    assert set(S(9, 4096, 16, 1).plan8()) == {"gate", "dx", "dw"}
    assert S(0, 16, 16, 4).plan8() == {}
    for bad in (S(-1, 16, 16, 4), S(9, 0, 16, 4)):
        with pytest.raises(dp.DeepmdException):
            bad.plan8()
    with pytest.raises(dp.DeepmdException):
        S(9, 16, 16, 4).plan8(0)
