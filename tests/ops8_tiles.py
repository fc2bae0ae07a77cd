"""Sizes (rows, d_in, d_hidden, d_out) at which every tile of the products that only the gated block's gradients from
a checkpoint have runs, whole and in slices, with tiles wholly inside the output and on its edges: dh, and
the gate with its gradient, with up to four outputs too (test_ops8_tiles.py asks the library for the tiles;
test_gpu_ops8_tiles.py runs them). The first ones are heads on descriptors of a few cells, whose gates are sliced."""
HEADS = [(192, 1600, 240, 240), (192, 1600, 240, 1), (1000, 1600, 240, 1), (1000, 1600, 240, 3), (64, 2048, 96, 1)]
SIZES = {
    "f32": [(64, 16, 32, 8), (72, 464, 40, 424), (6249, 83, 33, 1103), (345, 17, 4447, 2), (26352, 16, 40, 48),
            (67, 921, 1543, 133), (161, 67, 2065, 1217), (67, 19, 17, 3), (91, 19, 17, 1), (73, 379, 17, 3),
            (9141, 19, 17, 1), (135, 17, 1461, 3), (149, 17, 5059, 1), (443, 21, 2119, 2), (6197, 1099, 17, 1),
            (8565, 961, 17, 71), (129, 2379, 697, 1), (515, 103, 5947, 4), (7168, 16, 1056, 376),
            (208, 2672, 3096, 8), (75, 359, 17, 117), (6349, 2711, 123, 4), (1136, 864, 232, 8),
            (136, 1240, 1456, 24), (400, 104, 7680, 8), (3875, 1057, 939, 1), (496, 152, 2112, 4032),
            (345, 3349, 2099, 4)],
    "16": [(67, 19, 33, 7), (80, 928, 32, 800), (203, 19, 6535, 2), (2703, 17, 5807, 3), (80, 120, 6488, 2280),
           (65, 1677, 2385, 57), (65, 19, 19, 1), (81, 19, 19, 2), (71, 815, 19, 1), (129, 23, 4257, 1),
           (7003, 17, 101, 2), (25456, 32, 200, 200), (12115, 17, 589, 1), (30789, 17, 227, 4),
           (131, 1933, 1413, 4), (5449, 347, 535, 1), (72, 16, 16, 8), (65, 905, 21, 29), (65, 19, 6471, 2),
           (840, 16, 1464, 8), (8569, 2779, 81, 1), (271, 2467, 3269, 21), (72, 2936, 1648, 32),
           (27251, 1699, 73, 2), (6264, 136, 168, 3984), (480, 3376, 4104, 8), (2343, 3615, 845, 2),
           (272, 2960, 3520, 8), (2995, 3447, 665, 5), (577, 77, 6783, 3943)],
}
NEW = ("gate", "gate_back", "gate_outs", "gate_one", "dh")


def variants(dp, dtype, n, d, f, o):
    """{(product, tile rows, tile columns, sliced)} of a call of these sizes, the same with a tile wholly inside (and for
    the gate's gradient whether rows are whole chunks), and which of gate and dh are sliced together."""
    plan = dp.ops.GatedShape(n, d, f, o, dtype=dtype).plan8()
    whole = all(v % 8 == 0 for v in (n, d, f, o))
    seen = set()
    for what in NEW:
        if what in plan:
            rows, cols, slices = plan[what]
            tile = (what, rows, cols, slices > 1)
            seen.add(tile)
            if n >= rows and f >= (cols if what == "dh" else cols // 2):
                seen.add(tile + (whole if what == "gate_back" else None, "inside"))
    if "dh" in plan:
        seen.add(("gate_back", plan["gate_back"][2] > 1, "dh", plan["dh"][2] > 1))
    return seen
