"""Sizes beyond a C integer reach the operators as refused ones, not as their lower bits."""
import pytest


class Recorded:
    """Takes the library's place: keeps the arguments of the last call."""

    def __init__(self):
        self.args = None

    def __getattr__(self, name):
        def call(*args):
            self.args = args
            return 0
        return call


def test_shape(dp):
    S = dp.ops.GatedShape
    assert S(7, 3, 5, 2).saved_bytes() == 8 * 7 * 5
    for bad in (S(7, 3, 2 ** 32 + 5, 2), S(7, 2 ** 32 + 3, 5, 2), S(7, 3, 5, 2 ** 32 + 2), S(2 ** 64 + 7, 3, 5, 2),
                S(7, 3, 5, 2, ld_x=2 ** 64), S(7, 3, 5, 2, ld_down=2 ** 64 + 2), S(7, 3, 5, 2, dtype=2 ** 32),
                S(7, 3, 5, 2, act=2 ** 32 + 1)):
        assert bad.saved_bytes() == 0
    with pytest.raises(TypeError):
        S(7.5, 3, 5, 2)


@pytest.mark.parametrize("call", ["embed", "embed_grad"])
def test_lookup(dp, call):
    ops = object.__new__(dp.ops.Operators)
    ops._h, ops._lib, ops._error = 1, Recorded(), dp.DeepmdException
    run = getattr(ops, call)
    try:
        run(16, 16, 16, 4, 5, 8)
        assert ops._lib.args[1:5] == (0, 4, 5, 8)
        for args in ((2 ** 64 + 4, 5, 8), (4, 2 ** 32 + 5, 8), (4, 5, 2 ** 32 + 8), (4, -5, 8),
                     (4, 5, 8, "f32", 1.0, 2 ** 64 + 8), (4, 5, 8, "f32", 1.0, 0, 2 ** 64 + 8)):
            run(16, 16, 16, *args)
            assert ops._lib.args[2] == -1  # (n, which the library refuses)
        run(16, 16, 16, 4, 5, 8, 2 ** 32)
        assert ops._lib.args[1] == -1
    finally:
        ops._h = None
