"""Products that reach every kernel of hh_linear on 256 CUs, and what they
launch.  m, n and k are ragged as far as a kernel takes them so, the steps of
k that a tile takes are odd in number, and n is a multiple of 4 (an epilogue
of 4 values at a time) or not."""

# tiles straight to LDS: W's side, x's side
LARGE = [
    (33, 42, 192, 128, 64, 1), (35, 44, 192, 128, 64, 1), (34, 41, 2176, 128, 64, 12), (34, 40, 2240, 128, 64, 12),
    (129, 10967, 192, 128, 128, 1), (150, 11352, 192, 128, 128, 1), (1099, 42, 2752, 128, 128, 15),
    (1118, 40, 2816, 128, 128, 15),
    (717, 10866, 576, 128, 256, 1), (1191, 6476, 576, 128, 256, 1), (2246, 41, 4736, 128, 256, 15),
    (2186, 40, 4736, 128, 256, 15),
    (275, 10986, 192, 256, 128, 1), (1028, 3588, 192, 256, 128, 1), (33, 4257, 4544, 256, 128, 15),
    (34, 4196, 4416, 256, 128, 14),
    (1668, 4747, 192, 256, 256, 1), (2635, 3120, 192, 256, 256, 1), (131, 11051, 5248, 256, 256, 4),
    (130, 10924, 5760, 256, 256, 4),
]
# tiles through registers: the side of the tile
ANY = [
    (72, 42, 131, "same", 64, 1), (75, 40, 153, "same", 64, 1), (68, 41, 2115, "same", 64, 12), (68, 40, 2236, "same", 64, 12),
    (67, 8573, 141, "same", 128, 1), (76, 8764, 176, "same", 128, 1), (586, 66, 2364, "same", 128, 13),
    (67, 540, 2697, "same", 128, 15),
    (72, 42, 160, "int4", 64, 1), (68, 41, 2144, "int4", 64, 12), (67, 8573, 160, "int4", 128, 1),
    (586, 66, 2336, "int4", 128, 13), (67, 540, 2720, "int4", 128, 15),
    (72, 42, 131, "int4", 64, 1), (3, 41, 2115, "int4", 64, 12), (67, 8573, 141, "int4", 128, 1),
    (586, 66, 2364, "int4", 128, 13), (67, 540, 2697, "int4", 128, 15),
]
# few rows: tiles of 16 rows of x, of W, waves
ROWS = [
    (1, 8209, 416, "same", 1, 1, 4), (16, 8212, 1171, "same", 1, 1, 4), (17, 8209, 419, "same", 2, 2, 4),
    (32, 9000, 640, "same", 2, 2, 4), (33, 8209, 419, "same", 4, 2, 4), (64, 8230, 1155, "same", 4, 2, 4),
    (1, 8209, 416, "int4", 1, 2, 4), (9, 8212, 1184, "int4", 1, 2, 4), (20, 8209, 416, "int4", 2, 2, 4),
    (64, 8230, 1152, "int4", 4, 2, 4),
    (1, 8192, 1171, "same", 1, 1, 8), (31, 8180, 416, "same", 2, 1, 8), (50, 333, 1171, "same", 4, 1, 8),
    (16, 8179, 1184, "int4", 1, 1, 8), (19, 100, 2080, "int4", 2, 1, 8), (64, 8192, 416, "int4", 4, 1, 8),
]


def cases():
    """(m, n, k, weight, the kernel's mangled name with room for x's and y's types, splits, the grid's dimension of these)."""
    out = []
    for m, n, k, tn, tm, splits in LARGE:
        out.append((m, n, k, "same", f"linear_large_kernelILi%dELi%dELi{tn}ELi{tm}E", splits, 1))
    for m, n, k, weight, side, splits in ANY:
        mode = 0 if weight == "same" else 1 if k % 32 == 0 else 2
        out.append((m, n, k, weight, f"linear_tile_kernelILi%dELi%dELi{mode}ELi{side}E", splits, 2))
    for m, n, k, weight, mt, nt, waves in ROWS:
        out.append((m, n, k, weight, f"linear_rows_kernelILi%dELi%dELi{mt}ELi{nt}ELi{waves}ELb{int(weight == 'int4')}E", 1, 1))
    return out
