"""Gated products that reach every kernel of hh_gated_linear on 256 CUs, and
what they launch (both weights' rows count: n is half of a product's)."""

LARGE = [
    (33, 21, 192, 128, 64, 1), (35, 24, 192, 128, 64, 1), (34, 21, 2176, 128, 64, 12), (34, 20, 2240, 128, 64, 12),
    (129, 5483, 192, 128, 128, 1), (150, 5676, 192, 128, 128, 1), (2092, 46, 5184, 128, 128, 14), (1169, 20, 5696, 128, 128, 15),
    (717, 5437, 576, 128, 256, 1), (1191, 3236, 576, 128, 256, 1), (2062, 22, 7104, 128, 256, 16),
    (2156, 20, 6784, 128, 256, 16),
    (275, 5493, 192, 256, 128, 1), (1028, 1796, 192, 256, 128, 1), (33, 2097, 4672, 256, 128, 15),
    (34, 2100, 4416, 256, 128, 14),
    (1668, 2373, 192, 256, 256, 1), (2635, 1560, 192, 256, 256, 1), (131, 5529, 5248, 256, 256, 4),
    (130, 5464, 5760, 256, 256, 4),
]
ANY = [
    (72, 21, 131, "same", 64, 1), (75, 20, 153, "same", 64, 1), (68, 21, 2115, "same", 64, 12), (68, 20, 2236, "same", 64, 12),
    (67, 4287, 141, "same", 128, 1), (76, 4380, 176, "same", 128, 1), (686, 35, 1650, "same", 128, 13),
    (67, 270, 2697, "same", 128, 15),
    (72, 21, 160, "int4", 64, 1), (68, 21, 2144, "int4", 64, 12), (67, 4287, 160, "int4", 128, 1),
    (688, 47, 1920, "int4", 128, 15), (67, 270, 2720, "int4", 128, 15),
    (72, 21, 131, "int4", 64, 1), (3, 21, 2115, "int4", 64, 12), (67, 4287, 141, "int4", 128, 1),
    (767, 45, 3414, "int4", 128, 14), (67, 270, 2697, "int4", 128, 15),
]
# few rows: tiles of 16 rows of x, waves
ROWS = [
    (1, 8209, 416, "same", 1, 4), (16, 8212, 1171, "same", 1, 4), (17, 8209, 419, "same", 2, 4), (64, 8230, 1155, "same", 4, 4),
    (9, 8212, 1184, "int4", 1, 4), (20, 8209, 416, "int4", 2, 4), (64, 8230, 1152, "int4", 4, 4),
    (1, 8192, 1171, "same", 1, 8), (31, 818, 416, "same", 2, 8), (50, 333, 1171, "same", 4, 8),
    (16, 819, 1184, "int4", 1, 8), (19, 100, 2080, "int4", 2, 8), (64, 812, 416, "int4", 4, 8),
]

# whole rounds of one shape, then the other columns in another: m, n, k, the first launch's shape and columns, the second's shape
TWO = [(1544, 5875, 448, (256, 256), 4608, (256, 128)), (1562, 5278, 320, (256, 256), 4608, (128, 128)),
       (1429, 5496, 256, (256, 256), 5376, (128, 64)), (1538, 4997, 896, (256, 128), 4992, (128, 64))]


def cases():
    """(m, n, k, weight, the kernel's mangled name with room for x's and y's types, splits, the grid's dimension of these)."""
    out = []
    for m, n, k, tn, tm, splits in LARGE:
        out.append((m, n, k, "same", f"gated_large_kernelILi%dELi%dELi{tn}ELi{tm}E", splits, 1))
    for m, n, k, weight, side, splits in ANY:
        mode = 0 if weight == "same" else 1 if k % 32 == 0 else 2
        out.append((m, n, k, weight, f"gated_tile_kernelILi%dELi%dELi{mode}ELi{side}E", splits, 2))
    for m, n, k, weight, mt, waves in ROWS:
        out.append((m, n, k, weight, f"gated_rows_kernelILi%dELi%dELi{mt}ELi2ELi{waves}ELb{int(weight == 'int4')}E", 1, 1))
    return out
