"""Sizes that meet every kernel of the MX products (``kernels.mx_plan``): test_mx_plan.py holds that they do, the GPU tests
run them. Rows, columns and reductions are no multiples of a tile, of a step or of 32 where the kernel allows it."""

# Output tiles as (rows, weight rows, steps in the ring).
TILES = [(64, 128, 4), (128, 128, 3), (128, 256, 4), (192, 256, 3), (256, 256, 3), (32, 64, 4), (128, 256, 2), (64, 128, 2)]
SPLIT_TILES = TILES[:5]

# (tile, rows, columns, reduction) of whole tiles with columns by eights (16-byte stores) ...
WIDE = [(0, 79, 144, 1056), (1, 1839, 1064, 992), (2, 2236, 2872, 1312), (3, 2708, 3352, 1056), (4, 4554, 2616, 800), (5, 67, 80, 64),
        (6, 1482, 14680, 64), (7, 66, 136, 160)]
# ... and not; of split reductions with either. Both formats of the rows, but where one is named.
ODD = [(0, 73, 143, 1088), (1, 1552, 1281, 928), (2, 2049, 3463, 1056), (3, 2790, 3459, 928), (4, 2522, 4619, 800), (5, 65, 68, 64),
       (6, 5885, 3764, 64), (7, 73, 132, 160)]
SPLIT = [(0, 68, 136, 1952), (0, 66, 137, 1824), (1, 1414, 400, 7840), (1, 449, 1300, 7264), (2, 534, 2232, 9504), (2, 665, 1820, 10048),
         (3, 2817, 784, 12992), (3, 2723, 791, 10912)]
SPLIT_OF = {"e4m3": [(4, 501, 5696, 23840)], "e2m1": [(4, 2716, 1464, 8384), (4, 1841, 2247, 8896)]}

# The stream, (rows it holds, weight rows of a workgroup, waves), rows, columns, reduction: twelve waves from 96 steps of 128
# on, eight up to 95.
STREAM = [((16, 16, 12), 1, 3584, 18944), ((16, 16, 12), 1, 4096, 14336), ((16, 16, 12), 5, 33, 12320), ((16, 16, 8), 3, 1001, 12160),
          ((16, 16, 12), 3, 1001, 12192), ((16, 32, 8), 1, 5120, 13824), ((16, 32, 8), 2, 8190, 2080), ((16, 64, 8), 5, 8424, 1056),
          ((16, 64, 8), 15, 9001, 1376), ((32, 16, 8), 31, 3000, 1376), ((32, 32, 8), 24, 4217, 1376), ((64, 16, 8), 50, 1003, 1376),
          ((64, 16, 8), 64, 3584, 3584)]
STREAM_OF = {"e4m3": [], "e2m1": [((16, 16, 12), 16, 3584, 18944), ((32, 16, 12), 17, 1496, 12928), ((64, 16, 12), 37, 3472, 14080)]}

# The gate/up product: tile, rows, intermediate size, reduction. (The second and third tiles are only taken in splits with
# e4m3 rows.)
GATE_UP = [(0, 66, 96, 1248), (3, 1317, 4544, 1312), (4, 3361, 1824, 1568), (6, 1237, 8800, 64), (7, 65, 96, 160)]
GATE_UP_SPLIT = [(0, 81, 96, 1824), (1, 853, 736, 7072), (2, 1062, 608, 9568), (3, 554, 2336, 14752), (4, 385, 2848, 11968)]
GATE_UP_OF = {"e4m3": [(5, 23, 32, 1056), (5, 29, 18944, 3584)],
              "e2m1": [(1, 1271, 800, 416), (2, 2062, 1888, 672), (5, 29, 18944, 3584)]}
GATE_UP_STREAM = [(8, 1, 480, 1536), (8, 16, 8960, 1536), (3, 5, 96, 288)]  # waves, rows, intermediate size, reduction


def linear(fmt):
    """(plan, rows, columns, reduction) of every kernel of mx_linear; plan as in ``kernels.MXPlan`` without the splits."""
    return ([(TILES[t], False, *size) for t, *size in WIDE + ODD]
            + [(TILES[t], True, *size) for t, *size in SPLIT + SPLIT_OF[fmt]]
            + [((rows, cols, 0), waves, *size) for (rows, cols, waves), *size in STREAM + STREAM_OF[fmt]])


def gate_up(fmt):
    return ([(TILES[t], False, *size) for t, *size in GATE_UP + GATE_UP_OF[fmt]]
            + [(TILES[t], True, *size) for t, *size in GATE_UP_SPLIT]
            + [((16, 64, 0), waves, *size) for waves, *size in GATE_UP_STREAM])


def every(kind):
    return [(fmt, *case) for fmt in ("e4m3", "e2m1") for case in kind(fmt)]


def is_plan(plan, shape, detail):
    """Whether plan is the kernel that a case names."""
    if tuple(plan[:3]) != shape:
        return False
    return plan.splits_or_waves == detail if shape[2] == 0 else (plan.splits_or_waves > 1) == detail
