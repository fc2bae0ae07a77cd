"""Group norm of no rows, each of them a frame by itself: as many frames as rows is none."""
import ctypes as C

import pytest


@pytest.fixture()
def handle(dp):
    L, h = dp.lib(), C.c_void_p()
    L.dp_ops_create(0, C.byref(h))
    yield L, h
    L.dp_ops_destroy(h)


def test_no_rows_and_no_frames(dp, handle):
    L, h = handle
    shape = dp.ops.NormShape(0, 32, 4, frames=0)
    assert L.dp_group_norm(h, C.byref(shape.c), None, None, None, None, None, None, None) == 0
    assert L.dp_group_norm_grad(h, C.byref(shape.c), *[None] * 11) == 0


@pytest.mark.parametrize("rows,frames", [(8, 0), (0, -1), (8, -8)])
def test_frames_that_are_refused(dp, handle, rows, frames):
    L, h = handle
    shape = dp.ops.NormShape(rows, 32, 4, frames=1)
    shape.c.frames = frames
    for starts in (None, 4096):
        assert L.dp_group_norm(h, C.byref(shape.c), 4096, starts, None, None, 8192, None, None) == -1
        assert b"frames" in L.dp_ops_last_error(h)
