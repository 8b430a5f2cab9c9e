"""(m, n, k) of gated products whose gradients reach every kernel, tile shape
and split of hh_gated_linear_backward on 256 CUs; m and n end inside a step of
64, k is a multiple of 8 (tiles straight to LDS) or odd."""

SHAPES = [
    (9, 9, 16), (9, 10, 9), (9, 194, 9), (9, 321, 16), (9, 643, 4104), (9, 4294, 136), (9, 4455, 65), (9, 5492, 264),
    (9, 5596, 648), (10, 5478, 560), (133, 11, 5483), (402, 9, 9), (478, 1063, 9), (643, 9, 16), (778, 9, 4696),
    (1563, 1232, 16), (1572, 588, 16), (2061, 202, 9), (2433, 9, 3136), (2465, 385, 16), (3092, 4116, 136), (3604, 9, 2208),
    (4113, 458, 16), (4188, 3073, 136), (4561, 1029, 136), (5470, 10, 272),
]
# mangled names: the type, transposed on both sides (the weights' gradients) or not, the tile
TILES = [(256, 256), (256, 128), (128, 256), (128, 128), (128, 64)]
KERNELS = [f"gated_back_kernelILi2ELb{turn}ELi{c}ELi{r}E" for turn in (0, 1) for c, r in TILES] + \
          [f"gated_back_any_kernelILi2ELb{turn}ELi{s}E" for turn in (0, 1) for s in (128, 64)]
