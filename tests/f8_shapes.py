"""Shapes that reach each kernel of the products of the 8-bit floating tier, on 256 CUs. test_f8_coverage.py holds them to the
rules of csrc/kxw4_f8_route.hpp; the GPU tests of test_gpu_f8_tiles.py and test_gpu_f8_stream.py run them."""

CUS = 256

# A tile by tokens x weight rows, "parts" with the sum over the columns split: kernel -> shapes (T, K, the weights' M).
# K up to 14,992: 118 blocks, within what f8_ref.exact_weight's inputs may hold (118 * 35,295 < 2^22).
DENSE_BF16 = {
    "256x256": [(2100, 144, (5136,)), (4100, 272, (8208,)), (3100, 16, (4112,)), (1500, 400, (272, 16, 1040, 4112))],
    "256x256 parts": [(520, 14992, (5136,))],
    "256x128": [(1030, 1168, (4112,)), (700, 656, (272, 16, 1040, 4112))],
    "256x128 parts": [(700, 8208, (1040,)), (512, 14992, (5120,))],
    "128x128": [(520, 2064, (4112,)), (700, 144, (5136,))],
    "128x128 parts": [(1300, 4112, (528,))],
    "64x128": [(700, 640, (2064,)), (1024, 1024, (1024,))],
    "64x128 parts": [(130, 4112, (2064,)), (256, 8192, (512,))],
}
DENSE_F32 = {
    "128x128": [(2100, 144, (5136,)), (4100, 272, (8208,)), (1030, 1168, (4112,)), (1500, 400, (272, 16, 1040, 4112))],
    "128x128 parts": [(1030, 8208, (2064,))],
    "64x128": [(520, 2064, (4112,)), (700, 640, (2064,)), (700, 656, (272, 16, 1040, 4112))],
    "64x128 parts": [(130, 4112, (2064,)), (256, 8192, (512,))],
}
# (the choice's numbers: kernel -> id of kxw4_f8_route.hpp)
BF16_TILES = {"256x256": 0, "256x128": 1, "128x128": 2, "64x128": 3}
F32_TILES = {"128x128": 4, "64x128": 5}

# By group, of either output: run length -> shapes (T, k, groups, K, the weights' M)
GROUPED = {
    "short": [(300, 4, 20, 656, (1040,)), (700, 4, 100, 656, (1040,)), (1025, 3, 40, 16, (4112,)), (300, 4, 20, 656, (272, 1040))],
    "long": [(700, 4, 20, 656, (1040,)), (2300, 4, 70, 400, (272,)), (2600, 2, 40, 16, (2064,)), (700, 4, 20, 656, (272, 16, 1040, 400))],
}
# Weights past 2^32 bytes, by group: groups, K, M, and the rows of one slot each that make their runs short or long
PAST_32 = (70, 16384, 4096, {"short": 1200, "long": 9000})

# The kernel for few rows: rows of a tile, row-groups and waves of a work-group -> shapes (T, k, groups, K, the weights' M),
# groups 0 for one weight
STREAM = {
    (16, 1, 4): [(1, 1, 0, 400, (272,)), (16, 1, 0, 1040, (144, 272)), (5, 2, 9, 400, (144,)), (16, 1, 0, 8208, (272,))],
    (16, 2, 4): [(1, 1, 0, 400, (4112,)), (15, 1, 0, 528, (4112, 4240)), (9, 1, 0, 2064, (8208,)), (8, 1, 0, 5136, (8208, 16, 4112)),
                 (7, 4, 30, 400, (272,)), (60, 8, 64, 1040, (528, 272))],
    (16, 2, 8): [(13, 1, 0, 8208, (4112,)), (1, 1, 0, 14992, (5136,)), (4, 2, 8, 8208, (528,)), (16, 1, 16, 8192, (256,))],
    (32, 1, 4): [(33, 1, 0, 400, (272,)), (17, 1, 0, 2064, (1040,)), (50, 2, 3, 336, (272,))],
    (32, 2, 4): [(130, 1, 0, 400, (1040,)), (97, 1, 0, 1456, (2064,)), (100, 3, 5, 400, (528,)), (100, 3, 5, 400, (528, 16, 272))],
}


def cases(table):
    """(kernel, *shape) of every shape of a table."""
    return [(kernel, *shape) for kernel, shapes in table.items() for shape in shapes]
