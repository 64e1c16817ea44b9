"""Shapes of attention over shared keys in tiles of 32 and 128 rows: what the host test holds against
the library's choice and the GPU tests run.

Each: heads, kv heads, page, sizes of the groups, shared rows of each group, each sequence's own rows,
its query rows.  The tiles follow from the rows of q, the sequences and the groups alone."""


def spread(n, lo, hi):
    """n numbers from lo to hi, in no order."""
    return [lo + (7 * i + 3 * (i // 5)) % (hi - lo + 1) for i in range(n)]


# Rests and groups in one launch of tiles of 32 (a group of 128 to 511 rows a kv head on average).
TILES_32 = {
    # the last tile of a group full, of 8 rows, of 22, of 16
    "whole_tiles": (8, 1, 32, [40], [300], spread(40, 1, 40), [1] * 40),
    "two_groups": (16, 2, 64, [20, 25], [333, 1000], spread(45, 1, 70), [1] * 45),
    "odd_ratio": (5, 1, 32, [30], [97], spread(30, 1, 33), [1] * 30),
    "several_kv_heads": (24, 3, 128, [16, 18, 20], [640, 129, 500], spread(54, 1, 130), [1] * 54),
    # blocks of two rows, which see less than all of their own
    "blocks": (8, 1, 32, [12, 12], [250, 64], spread(24, 2, 50), [2] * 24),
    # rows of 1 to 4 tokens, idle sequences at both ends and between
    "ragged": (4, 1, 32, [30, 30], [200, 515], spread(60, 4, 40), [0] + spread(58, 0, 4) + [0]),
    # nothing of their own (without causal every key is a group's), and not all of them
    "no_rests": (8, 1, 32, [20], [128], [0] * 20, [1] * 20),
    "few_rests": (8, 1, 64, [24], [256], [5 if i % 6 == 1 else 0 for i in range(24)], [1] * 24),
    # groups of one block, of which a worker has many whole; a long one, cut among many workers
    "short": (64, 8, 32, [30, 31, 29], [32, 32, 64], spread(90, 1, 3), [1] * 90),
    "long": (8, 1, 64, [33], [9000], spread(33, 1, 20), [1] * 33),
    # a group that shares nothing among those that do
    "nothing_shared": (16, 1, 32, [10, 12, 11], [20, 400, 0], spread(33, 1, 50), [1] * 33),
}

# Groups in a launch of tiles of 128, rests in one of tiles of 16 (512 rows and more).
TILES_128 = {
    "whole_tiles": (8, 1, 32, [80], [300], spread(80, 1, 40), [1] * 80),
    "two_groups": (16, 2, 64, [70, 81], [333, 1000], spread(151, 1, 70), [1] * 151),
    "odd_ratio": (5, 1, 32, [107], [97], spread(107, 1, 33), [1] * 107),
    "blocks": (4, 1, 32, [40, 50], [250, 64], spread(90, 4, 50), [4] * 90),
    "sixteen_rows": (32, 2, 128, [36], [700], spread(36, 1, 140), [1] * 36),
    "ragged": (4, 1, 32, [100, 110], [200, 515], spread(210, 5, 40), [0] + spread(208, 1, 5) + [0]),
    "no_rests": (16, 1, 32, [40], [128], [0] * 40, [1] * 40),
    "few_rests": (8, 1, 64, [70], [256], [5 if i % 6 == 1 else 0 for i in range(70)], [1] * 70),
    "short": (64, 8, 32, [70, 66], [32, 96], spread(136, 1, 3), [1] * 136),
    "long": (8, 1, 64, [66], [9000], spread(66, 1, 20), [1] * 66),
    "nothing_shared": (16, 1, 32, [50, 40, 60], [20, 400, 0], spread(150, 1, 50), [1] * 150),
}
