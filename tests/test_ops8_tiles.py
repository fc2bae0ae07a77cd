"""The sizes of ops8_tiles.py reach every tile that the library takes for a product of the gated block's gradients from
a checkpoint on 256 compute units, whole and sliced (what it takes is asked of it for shapes drawn over the range)."""
import math
import os
import random
import re
import shutil
import subprocess

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


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gates_that_no_join_follows(dp, dtype):
    """The gate that sums h dy in its tiles is never sliced, and has no tile of 128 x 128 with two to four outputs."""
    rng = random.Random(1)
    for _ in range(5000):
        n, d, f = (round(math.exp(rng.uniform(0, math.log(m)))) for m in (100000, 4096, 8192))
        plan = dp.ops.GatedShape(n, d, f, rng.randint(1, 4), dtype=dtype).plan8()
        assert plan.get("gate_outs", (0, 0, 1))[2] == plan.get("gate_one", (0, 0, 1))[2] == 1
        assert plan.get("gate_outs", (0, 0, 1))[:2] != (128, 128)


def test_no_join_is_built_for_them(dp):
    """A kernel that no call may reach is not in the library (kEpiGateOuts is 6, kEpiGateOne 7)."""
    if not (shutil.which("nm") and os.path.exists(dp.LIB_PATH)):
        pytest.skip("no nm, or the library is not built")
    names = subprocess.run(["nm", "-C", dp.LIB_PATH], check=True, capture_output=True, text=True).stdout
    built = {m for m in re.findall(r"k_join<(\d), (\d)>", names)}
    assert {("0", "1"), ("0", "2"), ("0", "5")} <= built
    assert not [b for b in built if b[1] in "67"]


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
