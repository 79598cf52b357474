"""Sizes (M, K, N) of products with block-scaled 8-bit weights, by the tile and the parts of the sum that they take: every kind, whole and
partial along every side, with one block of 128 along the sum and with many."""

TILES = {
    (17, 128, 8): ("64", 1),
    (17, 128, 5120): ("64", 1),
    (300, 16, 5128): ("64", 1),
    (129, 2064, 5000): ("64", 1),
    (40, 5120, 640): ("64", 8),
    (70, 5136, 1032): ("64", 7),
    (700, 128, 4104): ("128 deep", 1),
    (500, 272, 5128): ("128 deep", 1),
    (500, 1040, 5128): ("128 deep", 1),
    (1500, 400, 5128): ("128 deep", 1),
    (333, 4112, 5096): ("128 deep", 2),
    (200, 5120, 5064): ("128 deep", 3),
    (1000, 1040, 5120): ("128", 1),
    (999, 2064, 5128): ("128", 1),
    (2000, 528, 5000): ("256", 1),
    (4100, 256, 4360): ("256", 1),
}
