"""Operators of trainable heads on device memory: embedding lookup and its gradient, and
the gated feed-forward block, forward and backward (the dp_ops part of
include/dp_amd.h). As the device entry points of `DeepPot`, every array is a raw
device pointer (an int), and work is ordered on `stream`; unlike the synchronous ones
the calls return without waiting. Failures raise DeepmdException. Ids are 32-bit integers (int32): a
pointer to torch's int64 indices is read as pairs of them.
"""
from __future__ import annotations

import ctypes as C

TYPE_F32, TYPE_BF16, TYPE_F16 = 0, 1, 2
ACT_TANH, ACT_SILU, ACT_GELU = 0, 1, 2
TYPES = {"f32": TYPE_F32, "bf16": TYPE_BF16, "f16": TYPE_F16}
ACTS = {"tanh": ACT_TANH, "silu": ACT_SILU, "gelu": ACT_GELU}

EXPORTED = ("dp_ops_create", "dp_ops_destroy", "dp_ops_last_error", "dp_ops_device_bytes", "dp_embed",
            "dp_embed_grad", "dp_gated_saved_bytes", "dp_gated_forward", "dp_gated_backward", "dp_debug_gated_plan")
PRODUCTS = ("gate", "down", "gate_grad", "dx", "dw", "dw_down")


class _Shape(C.Structure):
    _fields_ = [("rows", C.c_int64), ("d_in", C.c_int), ("d_hidden", C.c_int), ("d_out", C.c_int),
                ("type", C.c_int), ("act", C.c_int), ("ld_x", C.c_int64), ("ld_y", C.c_int64),
                ("ld_hidden", C.c_int64), ("ld_down", C.c_int64)]


def bind(L):
    """Argument types of the dp_ops entry points."""
    P, I, N = C.c_void_p, C.c_int, C.c_int64
    S = C.POINTER(_Shape)
    L.dp_ops_create.argtypes = [I, C.POINTER(P)]
    L.dp_ops_destroy.argtypes = [P]
    L.dp_ops_destroy.restype = None
    L.dp_ops_last_error.argtypes = [P]
    L.dp_ops_last_error.restype = C.c_char_p
    L.dp_ops_device_bytes.argtypes = [P]
    L.dp_ops_device_bytes.restype = C.c_size_t
    L.dp_embed.argtypes = [P, I, N, I, I, P, P, N, C.c_float, P, N, P]
    L.dp_embed_grad.argtypes = [P, I, N, I, I, P, P, N, C.c_float, P, N, P]
    L.dp_gated_saved_bytes.argtypes = [S]
    L.dp_gated_saved_bytes.restype = C.c_size_t
    L.dp_debug_gated_plan.argtypes = [S, I, C.POINTER(C.c_int)]
    L.dp_gated_forward.argtypes = [P, S, P, P, P, P, P, P, P]
    L.dp_gated_backward.argtypes = [P, S, P, P, P, P, P, P, P, P, P, P, P]


# ctypes drops the upper bits of what a C integer does not hold: such sizes are passed on as -1, which every
# call refuses (one test of several together: a call on few rows takes as long as its Python).
def _code(names, v):
    return names.get(v, -1) if isinstance(v, str) else -1 if v >> 31 else int(v)


class GatedShape:
    """Sizes, type, activation and row lengths (0: packed) of a gated block
    (dp_gated_shape). `dtype` "f32", "bf16" or "f16"; `act` "tanh", "silu" or "gelu"."""

    def __init__(self, rows, d_in, d_hidden, d_out, dtype="f32", act="silu", ld_x=0, ld_y=0, ld_hidden=0,
                 ld_down=0):
        if (d_in | d_hidden | d_out) >> 31:
            d_in = -1
        if (rows | ld_x | ld_y | ld_hidden | ld_down) >> 63:
            rows = -1
        self.c = _Shape(rows, d_in, d_hidden, d_out, _code(TYPES, dtype), _code(ACTS, act), ld_x, ld_y, ld_hidden,
                        ld_down)

    def saved_bytes(self) -> int:
        """Bytes that gated_forward keeps for gated_backward (dp_gated_saved_bytes)."""
        from . import lib
        return int(lib().dp_gated_saved_bytes(C.byref(self.c)))

    def plan(self, compute_units: int = 256) -> dict:
        """{product: (tile rows, tile columns, slices)} of those that run as tiles (dp_debug_gated_plan)."""
        from . import DeepmdException, lib
        p = (C.c_int * (3 * len(PRODUCTS)))()
        if lib().dp_debug_gated_plan(C.byref(self.c), compute_units, p) != 0:
            raise DeepmdException("dp_debug_gated_plan: a shape that the calls refuse")
        return {k: tuple(p[3 * i:3 * i + 3]) for i, k in enumerate(PRODUCTS) if p[3 * i]}


class Operators:
    """A handle of the operators on one GPU (dp_ops)."""

    def __init__(self, gpu_rank: int = 0):
        from . import DeepmdException, lib
        self._h = None
        self._lib, self._error = lib(), DeepmdException
        h = C.c_void_p()
        rc = self._lib.dp_ops_create(gpu_rank, C.byref(h))
        if rc != 0:
            msg = self._lib.dp_ops_last_error(h).decode() if h else "dp_ops_create failed"
            self._lib.dp_ops_destroy(h)
            raise DeepmdException(f"dp_ops_create failed ({rc}): {msg}")
        self._h = h

    def __del__(self):
        if getattr(self, "_h", None):
            self._lib.dp_ops_destroy(self._h)
            self._h = None

    def _check(self, rc):
        if rc != 0:
            raise self._error(f"({rc}) {self._lib.dp_ops_last_error(self._h).decode()}")

    def embed(self, d_ids: int, d_table: int, d_out: int, n: int, vocab: int, width: int, dtype="f32",
              scale: float = 1.0, ld_table: int = 0, ld_out: int = 0, stream: int = 0):
        """out[i] = scale * table[ids[i]]; zeros for an id outside the table (dp_embed)."""
        if (vocab | width) >> 31 or (n | ld_table | ld_out) >> 63:
            n = -1
        self._check(self._lib.dp_embed(self._h, _code(TYPES, dtype), n, vocab, width, d_ids or None, d_table or None,
                                       ld_table, scale, d_out or None, ld_out, stream or None))

    def embed_grad(self, d_ids: int, d_dout: int, d_dtable: int, n: int, vocab: int, width: int, dtype="f32",
                   scale: float = 1.0, ld_dout: int = 0, ld_dtable: int = 0, stream: int = 0):
        """dtable[v] = scale * sum of dout[i] over ids[i] == v, every row written (dp_embed_grad)."""
        if (vocab | width) >> 31 or (n | ld_dout | ld_dtable) >> 63:
            n = -1
        self._check(self._lib.dp_embed_grad(self._h, _code(TYPES, dtype), n, vocab, width, d_ids or None,
                                            d_dout or None, ld_dout, scale, d_dtable or None, ld_dtable,
                                            stream or None))

    def gated_forward(self, shape: GatedShape, d_x: int, d_w_gate: int, d_w_up: int, d_w_down: int, d_y: int,
                      saved: int = 0, stream: int = 0):
        """y = (act(x w_gate) * (x w_up)) w_down; `saved` (shape.saved_bytes() bytes) keeps
        what the backward needs (dp_gated_forward)."""
        self._check(self._lib.dp_gated_forward(self._h, C.byref(shape.c), d_x or None, d_w_gate or None,
                                               d_w_up or None, d_w_down or None, d_y or None, saved or None,
                                               stream or None))

    def gated_backward(self, shape: GatedShape, d_x: int, d_w_gate: int, d_w_up: int, d_w_down: int, saved: int,
                       d_dy: int, d_dx: int = 0, d_dw_gate: int = 0, d_dw_up: int = 0, d_dw_down: int = 0,
                       stream: int = 0):
        """The gradients of x and of the weights from dy (dp_gated_backward); an output
        given as 0 is not formed."""
        self._check(self._lib.dp_gated_backward(self._h, C.byref(shape.c), d_x or None, d_w_gate or None,
                                                d_w_up or None, d_w_down or None, saved or None, d_dy or None,
                                                d_dx or None, d_dw_gate or None, d_dw_up or None,
                                                d_dw_down or None, stream or None))

    def device_bytes(self) -> int:
        """Peak device bytes of the handle's workspaces."""
        return int(self._lib.dp_ops_device_bytes(self._h))
