"""Calls and the variant of a kernel that each is for: the plans say so on the
CPU (test_variants.py), the values are checked on the GPU
(test_gpu_variants.py). A plan that is fitted anew and sends a call elsewhere
fails the first, so that no variant goes untested."""
from __future__ import annotations

SPLIT, PAIR = 0, 1  # a product by single CTAs, by pairs

# tokens, rows, cols, bias, add (2: y itself), values between rows of y; kernel, tokens a tile, CTAs (pairs) that split a
# tile's columns, panels of a stage, tiles
LINEAR = [
    # pairs that walk several tiles: two accumulators, the ring carried over, scales and added rows of the next tile;
    # ragged tokens and channels, tiles walked 32 together, more and fewer stages than a tile has
    (370, 27457, 515, 1, 0, 0, PAIR, 192, 1, 1, 216), (1277, 25872, 163, 0, 1, 0, PAIR, 256, 1, 1, 510),
    (1322, 12992, 370, 1, 2, 4, PAIR, 192, 1, 1, 357), (623, 25882, 426, 0, 2, 0, PAIR, 160, 1, 2, 408),
    (1030, 15865, 457, 1, 1, 1, PAIR, 160, 1, 2, 434), (312, 25614, 731, 0, 0, 3, PAIR, 160, 1, 2, 202),
    (1710, 6871, 524, 0, 1, 1, PAIR, 224, 1, 1, 216), (242, 21908, 1573, 1, 0, 0, PAIR, 128, 1, 2, 172),
    (300, 14413, 1429, 1, 1, 0, PAIR, 160, 1, 2, 114), (2682, 15813, 1799, 1, 2, 0, PAIR, 192, 1, 1, 868),
    (2000, 5000, 2400, 0, 1, 0, PAIR, 192, 1, 1, 220),
    # pairs that split a tile's columns
    (49, 6551, 15143, 1, 1, 1, PAIR, 64, 2, 2, 26), (2511, 142, 14188, 0, 2, 0, PAIR, 128, 3, 1, 20),
    (1904, 139, 19339, 1, 0, 2, PAIR, 128, 4, 1, 15),
    # single CTAs: whole columns, many tiles, and splits
    (4099, 6200, 300, 1, 2, 0, SPLIT, 240, 1, 1, 882), (300, 4096, 2560, 0, 1, 0, SPLIT, 80, 1, 2, 128),
    (53, 6961, 10665, 1, 1, 0, SPLIT, 64, 2, 1, 55), (2793, 17, 7489, 0, 1, 0, SPLIT, 64, 3, 1, 44),
    (1, 2912, 4032, 1, 2, 0, SPLIT, 16, 4, 2, 23), (31, 1000, 4096, 0, 1, 0, SPLIT, 16, 6, 2, 16),
    (333, 515, 9000, 1, 2, 1, SPLIT, 112, 8, 1, 15),
]

# the longest rows, all codes -128
LARGEST = [(20, 130, SPLIT), (200, 1500, PAIR)]

# one token among others, of the same weights: tokens from, to
BATCH = (6513, 2729)  # rows, cols
SLICES = [(0, 363, PAIR), (0, 1, SPLIT), (5, 21, SPLIT), (100, 164, SPLIT), (150, 305, SPLIT), (3, 363, PAIR)]

# products at once on two streams
TOGETHER = (27457, 515)
TOKENS = [(3, SPLIT), (370, PAIR)]

# rows of logits, vocabulary, top; threads of a CTA, loads ahead, CTAs that share a row
WIDE, NARROW = 512, 256
LOGPROBS = [
    (180, 16805, 0, WIDE, 1, 1), (145, 33049, 0, WIDE, 1, 2), (69, 66440, 0, WIDE, 1, 4), (3, 131216, 0, WIDE, 1, 8),
    (371, 8287, 0, NARROW, 1, 1), (560, 10019, 0, NARROW, 1, 1), (180, 216797, 0, NARROW, 1, 2),
    (85, 32795, 0, NARROW, 1, 4), (34, 67845, 0, NARROW, 1, 8),
    (601, 8249, 0, NARROW, 0, 1), (2004, 10441, 0, NARROW, 0, 1), (300, 16444, 0, NARROW, 0, 2),
    (154, 33361, 0, NARROW, 0, 4), (73, 66030, 0, NARROW, 0, 8),
    (149, 17364, 5, WIDE, 1, 1), (72, 33092, 20, WIDE, 1, 2), (32, 65614, 5, WIDE, 1, 4), (2, 131157, 32, WIDE, 1, 8),
    (298, 8208, 20, NARROW, 1, 1), (84, 131267, 5, NARROW, 1, 4), (34, 264053, 9, NARROW, 1, 8),
    (597, 8505, 5, NARROW, 0, 1), (300, 37896, 32, NARROW, 0, 2), (149, 83205, 1, NARROW, 0, 4),
    (74, 119467, 5, NARROW, 0, 8),
]
GROUPS = 3  # each thread meets so many of its groups of 16 logits
