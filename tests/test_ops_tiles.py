"""The sizes of ops_tiles.py reach every tile that the library takes for a product of the gated block
on 256 compute units (what it takes is asked of it for shapes drawn over the whole range)."""
import math
import random

import pytest

from ops_tiles import SIZES, variants


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_every_tile_is_run(dp, dtype):
    rng = random.Random(dtype)

    def size(lo, hi, whole):
        v = round(math.exp(rng.uniform(math.log(lo), math.log(hi))))
        return max(8, v // 8 * 8) if whole else v | 1

    taken = set()
    for _ in range(30000):
        whole = rng.random() < 0.5
        taken |= variants(dp, dtype, size(9, 100000, whole), size(16, 4096, whole), size(16, 8192, whole),
                          1 if rng.random() < 0.15 and not whole else size(8, 4096, whole))
    run = set().union(*(variants(dp, dtype, *s) for s in SIZES["f32" if dtype == "f32" else "16"]))
    assert {v[:4] for v in taken} <= {v[:4] for v in run}
    # with a tile wholly inside the output, wherever that happens, for odd rows and for whole chunks
    inside = {v for v in taken if v[4]}
    assert len(inside) > 60 and inside <= run


def test_plan(dp):
    S = dp.ops.GatedShape
    assert set(S(9, 16, 16, 5).plan()) == {"gate", "down", "gate_grad", "dx", "dw", "dw_down"}
    assert set(S(8, 16, 16, 5).plan()) == {"gate_grad", "dx", "dw", "dw_down"}
    assert set(S(9, 16, 16, 4).plan()) == {"gate", "dx", "dw"}
    assert S(0, 16, 16, 4).plan() == {}
    for bad in (S(-1, 16, 16, 4), S(9, 0, 16, 4)):
        with pytest.raises(dp.DeepmdException):
            bad.plan()
    with pytest.raises(dp.DeepmdException):
        S(9, 16, 16, 4).plan(0)
