"""Sizes (rows, d_in, d_hidden, d_out) at which every tile of every product of the gated block runs, whole
and in slices, with tiles wholly inside the output and on its edges, with rows of odd lengths
and of whole 16-byte chunks (test_ops_tiles.py asks the library for the tiles; test_gpu_ops_tiles.py runs them)."""
SIZES = {
    "f32": [(64, 2736, 72, 40), (71, 2805, 65, 41), (64, 32, 944, 1760), (65, 37, 1821, 909), (16403, 133, 33, 81),
            (10728, 160, 40, 144), (2496, 152, 632, 240), (3205, 163, 581, 183), (9207, 985, 17, 601),
            (8376, 856, 24, 864), (233, 2239, 1107, 2319), (136, 3200, 1384, 3320), (149, 59, 1521, 2761),
            (200, 48, 2208, 1504), (3123, 25, 3141, 489), (1728, 1496, 2168, 1216), (360, 4008, 1432, 1),
            (4199, 35, 361, 2807), (208, 1096, 4184, 4256), (3128, 3496, 256, 408), (14344, 1120, 248, 1),
            (1832, 16, 392, 3904), (6299, 237, 1269, 23)],
    "16": [(725, 145, 247, 51), (73, 1005, 807, 911), (64, 1008, 912, 960), (72, 40, 6360, 1808),
           (73, 2185, 2617, 4257), (7081, 215, 97, 233), (3640, 432, 16, 440), (136, 2088, 1680, 16),
           (20952, 24, 336, 352), (12991, 523, 241, 439), (6081, 1741, 19, 2393), (17512, 808, 136, 128),
           (135, 345, 8283, 1), (4341, 61, 3609, 533), (720, 2784, 1496, 1), (736, 40, 3232, 3040),
           (496, 3144, 2464, 16), (653, 3915, 3283, 3505), (6384, 400, 2808, 88), (705, 21, 6385, 3743),
           (2216, 16, 6472, 1176), (13880, 56, 416, 1040), (12949, 199, 571, 3431), (8792, 3416, 208, 40),
           (19912, 224, 280, 2144)],
}


def variants(dp, dtype, n, d, f, o):
    """{(product, tile rows, tile columns, sliced, a tile wholly inside, whole chunks)} of a step of these sizes.
    The two weight products are one kernel."""
    out = {"gate": (n, f), "down": (n, o), "gate_grad": (n, f), "dx": (n, d), "dw": (d, f), "dw_down": (f, o)}
    whole = all(v % 8 == 0 for v in (n, d, f, o))
    seen = set()
    for what, (rows, cols, slices) in dp.ops.GatedShape(n, d, f, o, dtype=dtype).plan().items():
        width = cols // 2 if what == "gate" else cols  # (a gate's tile holds as many columns of g as of u)
        inside = out[what][0] >= rows and out[what][1] >= width
        seen.add(("dw" if what == "dw_down" else what, rows, cols, slices > 1, inside, whole))
    return seen
