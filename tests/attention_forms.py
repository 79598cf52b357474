"""Sizes of attention over packed rows that take tiles of 32 rows with shared keys: rows of the requests, keys of the requests, rows
behind, heads, key heads, head_dim."""

SHARED = [
    ([1], [65], 0, 1, 1, 64),
    ([1], [512], 0, 40, 40, 128),
    ([16], [2000], 3, 40, 40, 128),
    ([3, 1, 9], [140, 0, 170], 4, 4, 2, 64),
    ([3, 1, 9], [140, 0, 170], 4, 4, 2, 128),
    ([32, 31, 33], [129, 127, 300], 1, 6, 2, 64),
    ([0, 40, 0, 27], [5, 163, 9, 264], 20, 3, 3, 128),
    ([100], [257], 29, 8, 8, 64),
    ([70, 1], [96, 70], 0, 40, 8, 128),
]
