"""Operators of trainable heads on device memory: embedding lookup and its gradient, the
gated feed-forward block, forward and backward, group norm with an activation, forward and
backward, checkpoints of activations in 8 bits with the gradients taken from them, and products in 8-bit
integers (the dp_ops part of include/dp_amd.h). As the device entry points of `DeepPot`, every array is a raw
device pointer (an int), and work is ordered on `stream`; unlike the synchronous ones
the calls return without waiting. Failures raise DeepmdException. Ids are 32-bit integers (int32): a
pointer to torch's int64 indices is read as pairs of them.
"""
from __future__ import annotations

import ctypes as C

TYPE_F32, TYPE_BF16, TYPE_F16 = 0, 1, 2
ACT_TANH, ACT_SILU, ACT_GELU, ACT_NONE = 0, 1, 2, 3
TYPES = {"f32": TYPE_F32, "bf16": TYPE_BF16, "f16": TYPE_F16}
ACTS = {"tanh": ACT_TANH, "silu": ACT_SILU, "gelu": ACT_GELU, "none": ACT_NONE}

EXPORTED = ("dp_ops_create", "dp_ops_destroy", "dp_ops_last_error", "dp_ops_device_bytes", "dp_embed",
            "dp_embed_grad", "dp_gated_saved_bytes", "dp_gated_forward", "dp_gated_backward", "dp_debug_gated_plan",
            "dp_keep8_bytes", "dp_keep8", "dp_restore8", "dp_gated_backward8", "dp_weights8", "dp_linear8",
            "dp_group_norm", "dp_group_norm_grad", "dp_debug_gated_plan8")
PRODUCTS = ("gate", "down", "gate_grad", "dx", "dw", "dw_down")
PRODUCTS8 = ("gate", "gate_back", "gate_outs", "gate_one", "dh", "dx", "dw", "dw_down")


class _Shape(C.Structure):
    _fields_ = [("rows", C.c_int64), ("d_in", C.c_int), ("d_hidden", C.c_int), ("d_out", C.c_int),
                ("type", C.c_int), ("act", C.c_int), ("ld_x", C.c_int64), ("ld_y", C.c_int64),
                ("ld_hidden", C.c_int64), ("ld_down", C.c_int64)]


class _Linear8(C.Structure):
    _fields_ = [("rows", C.c_int64), ("d_in", C.c_int), ("d_out", C.c_int), ("type", C.c_int), ("act", C.c_int),
                ("ld_x", C.c_int64), ("ld_y", C.c_int64), ("ld_w", C.c_int64)]


class _Norm(C.Structure):
    _fields_ = [("rows", C.c_int64), ("channels", C.c_int), ("groups", C.c_int), ("frames", C.c_int),
                ("type", C.c_int), ("act", C.c_int), ("eps", C.c_float), ("ld_x", C.c_int64), ("ld_y", C.c_int64)]


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
    for plan in (L.dp_debug_gated_plan, L.dp_debug_gated_plan8):
        plan.argtypes = [S, I, C.POINTER(C.c_int)]
    L.dp_gated_forward.argtypes = [P, S, P, P, P, P, P, P, P]
    L.dp_gated_backward.argtypes = [P, S, P, P, P, P, P, P, P, P, P, P, P]
    L.dp_keep8_bytes.argtypes = [N, I]
    L.dp_keep8_bytes.restype = C.c_size_t
    L.dp_keep8.argtypes = [P, I, N, I, P, N, P, P]
    L.dp_restore8.argtypes = [P, I, N, I, P, P, N, P]
    L.dp_gated_backward8.argtypes = [P, S, P, P, P, P, P, P, P, P, P, P]
    L.dp_weights8.argtypes = [P, I, I, I, P, N, P, N, P, P]
    L.dp_linear8.argtypes = [P, C.POINTER(_Linear8), P, P, P, P, P, P, P]
    L.dp_group_norm.argtypes = [P, C.POINTER(_Norm), P, P, P, P, P, P, P]
    L.dp_group_norm_grad.argtypes = [P, C.POINTER(_Norm), P, P, P, P, P, P, P, P, P, P, P]


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
        return self._plan("dp_debug_gated_plan", PRODUCTS, compute_units)

    def plan8(self, compute_units: int = 256) -> dict:
        """The same of gated_backward8 (dp_debug_gated_plan8)."""
        return self._plan("dp_debug_gated_plan8", PRODUCTS8, compute_units)

    def _plan(self, call, products, compute_units):
        from . import DeepmdException, lib
        p = (C.c_int * (3 * len(products)))()
        if getattr(lib(), call)(C.byref(self.c), compute_units, p) != 0:
            raise DeepmdException(call + ": a shape that the calls refuse")
        return {k: tuple(p[3 * i:3 * i + 3]) for i, k in enumerate(products) if p[3 * i]}


class Linear8Shape:
    """Sizes, type, activation and row lengths (0: packed) of a product in 8-bit integers
    (dp_linear8_shape). `act` "none", "tanh", "silu" or "gelu"; `ld_w` in bytes."""

    def __init__(self, rows, d_in, d_out, dtype="f32", act="none", ld_x=0, ld_y=0, ld_w=0):
        if (d_in | d_out) >> 31:
            d_in = -1
        if (rows | ld_x | ld_y | ld_w) >> 63:
            rows = -1
        self.c = _Linear8(rows, d_in, d_out, _code(TYPES, dtype), _code(ACTS, act), ld_x, ld_y, ld_w)


class NormShape:
    """Sizes, type, activation, eps and row lengths (0: packed) of a group norm (dp_norm_shape): `groups` divides
    `channels`; `frames` equal parts of the rows, or as many as the starts given with the call name."""

    def __init__(self, rows, channels, groups, frames=1, dtype="f32", act="none", eps=1e-5, ld_x=0, ld_y=0):
        if (channels | groups | frames) >> 31:
            channels = -1
        if (rows | ld_x | ld_y) >> 63:
            rows = -1
        self.c = _Norm(rows, channels, groups, frames, _code(TYPES, dtype), _code(ACTS, act), eps, ld_x, ld_y)


def keep8_bytes(rows: int, cols: int) -> int:
    """Bytes of the 8-bit checkpoint of rows x cols values (dp_keep8_bytes)."""
    from . import lib
    return 0 if cols >> 31 or rows >> 63 else int(lib().dp_keep8_bytes(rows, cols))


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

    def keep8(self, d_x: int, kept: int, rows: int, cols: int, dtype="f32", ld_x: int = 0, stream: int = 0):
        """The 8-bit checkpoint of x [rows][cols] into `kept` (keep8_bytes(rows, cols) bytes; dp_keep8)."""
        if cols >> 31 or (rows | ld_x) >> 63:
            rows = -1
        self._check(self._lib.dp_keep8(self._h, _code(TYPES, dtype), rows, cols, d_x or None, ld_x, kept or None,
                                       stream or None))

    def restore8(self, kept: int, d_x: int, rows: int, cols: int, dtype="f32", ld_x: int = 0, stream: int = 0):
        """What a checkpoint holds, as x [rows][cols] (dp_restore8)."""
        if cols >> 31 or (rows | ld_x) >> 63:
            rows = -1
        self._check(self._lib.dp_restore8(self._h, _code(TYPES, dtype), rows, cols, kept or None, d_x or None, ld_x,
                                          stream or None))

    def gated_backward8(self, shape: GatedShape, kept: int, d_w_gate: int, d_w_up: int, d_w_down: int, d_dy: int,
                        d_dx: int = 0, d_dw_gate: int = 0, d_dw_up: int = 0, d_dw_down: int = 0, stream: int = 0):
        """gated_backward from the 8-bit checkpoint of x alone, at the values it restores; the
        forward keeps nothing (dp_gated_backward8)."""
        self._check(self._lib.dp_gated_backward8(self._h, C.byref(shape.c), kept or None, d_w_gate or None,
                                                 d_w_up or None, d_w_down or None, d_dy or None, d_dx or None,
                                                 d_dw_gate or None, d_dw_up or None, d_dw_down or None,
                                                 stream or None))

    def weights8(self, d_w: int, d_w8: int, d_scale: int, d_in: int, d_out: int, dtype="f32", ld_w: int = 0,
                 ld_w8: int = 0, stream: int = 0):
        """w [d_in][d_out] as rows of 8-bit integers, one for each output channel, d_w8 [d_out][ld_w8] (0: d_in up to
        a multiple of 16), and their scales, fp32 [d_out] (dp_weights8)."""
        if (d_in | d_out) >> 31 or (ld_w | ld_w8) >> 63:
            d_in = -1
        self._check(self._lib.dp_weights8(self._h, _code(TYPES, dtype), d_in, d_out, d_w or None, ld_w, d_w8 or None,
                                          ld_w8, d_scale or None, stream or None))

    def linear8(self, shape: Linear8Shape, d_x: int, d_w: int, d_w_scale: int, d_y: int, d_up: int = 0,
                d_up_scale: int = 0, stream: int = 0):
        """y = act(x w), or act(x w) * (x up), on 8-bit weights and the rows of x in 8 bits (dp_linear8)."""
        self._check(self._lib.dp_linear8(self._h, C.byref(shape.c), d_x or None, d_w or None, d_w_scale or None,
                                         d_up or None, d_up_scale or None, d_y or None, stream or None))

    def group_norm(self, shape: NormShape, d_x: int, d_gamma: int, d_beta: int, d_y: int, stats: int = 0,
                   starts: int = 0, stream: int = 0):
        """y = act(gamma (x - m) r + beta) with m and r of each frame and group, which `stats` (fp32
        [frames][groups][2]) keeps for the backward; `starts`: int32 [frames + 1], the frames' first rows
        (dp_group_norm)."""
        self._check(self._lib.dp_group_norm(self._h, C.byref(shape.c), d_x or None, starts or None, d_gamma or None,
                                            d_beta or None, d_y or None, stats or None, stream or None))

    def group_norm_grad(self, shape: NormShape, d_x: int, d_gamma: int, d_beta: int, stats: int, d_dy: int,
                        d_dx: int = 0, d_dgamma: int = 0, d_dbeta: int = 0, kept: int = 0, starts: int = 0,
                        stream: int = 0):
        """The gradients of x, gamma and beta (dp_group_norm_grad), at x or (d_x 0) at its checkpoint `kept`; an
        output given as 0 is not formed."""
        self._check(self._lib.dp_group_norm_grad(self._h, C.byref(shape.c), d_x or None, kept or None, starts or None,
                                                 d_gamma or None, d_beta or None, stats or None, d_dy or None,
                                                 d_dx or None, d_dgamma or None, d_dbeta or None, stream or None))

    def device_bytes(self) -> int:
        """Peak device bytes of the handle's workspaces."""
        return int(self._lib.dp_ops_device_bytes(self._h))
