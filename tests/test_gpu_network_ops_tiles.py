"""The products of a wider network's operators in every tile that they can
take: sizes that are no multiples of a tile's, with sums of several slices.
Which tile a size takes is asked of the library, so that another rule for it
cannot leave a kernel without a test.  References and tolerances:
test_gpu_network_ops.py."""
import ctypes
import os

import pytest
import torch

from hive_neuralnet_amd import hive_gpu
from test_gpu_network_ops import BF16, F16, F32, _check_gated, _gated, ext  # noqa: F401

KINDS = {F32: 0, F16: 1, BF16: 2}
# (rows * 1000 + columns) * 100 + stages * 10 + blocks of a compute unit
LARGE, ALONE, MIDDLE, SMALL = 25625621, 12812841, 12812822, 6406433  # 16 bits
WIDE, SMALL_FLOAT = 6412822, 6406432  # float32
# (rows, columns, hidden units): the tiles of h, dx and the weights' gradients of 16-bit tensors, and of float32
GATED = {
    (2999, 1237, 515): ((ALONE, ALONE, SMALL), (WIDE, WIDE, WIDE)),
    (513, 441, 6905): ((LARGE, ALONE, MIDDLE), None),
    (517, 448, 6912): ((LARGE, ALONE, MIDDLE), None),  # taken as they are
    (65, 1009, 8035): ((SMALL, MIDDLE, LARGE), None),
    (67, 1008, 8040): ((SMALL, MIDDLE, LARGE), None),
    (10941, 665, 201): ((MIDDLE, LARGE, ALONE), None),
    (10945, 664, 208): ((MIDDLE, LARGE, ALONE), None),
    (67, 130, 200): ((SMALL,) * 3, (SMALL_FLOAT,) * 3),
    (65, 441, 4145): ((SMALL, SMALL, MIDDLE), (WIDE, WIDE, SMALL_FLOAT)),
}


def _tiles(t, sizes):
    tiles = (ctypes.c_int * 3)()
    assert hive_gpu.load_library().hg_gated_tiles(KINDS[t], *sizes, tiles) == 0
    return tuple(tiles)


@pytest.mark.skipif(not os.path.exists(hive_gpu.LIB_PATH), reason="libhive_gpu.so not built")
def test_the_sizes_below_take_every_tile():
    for sizes, (half, full) in GATED.items():
        assert _tiles(F16, sizes) == _tiles(BF16, sizes) == half, sizes
        assert full is None or _tiles(F32, sizes) == full, sizes
    for product in range(3):
        assert {half[product] for half, _ in GATED.values()} == {LARGE, ALONE, MIDDLE, SMALL}, product
        assert {full[product] for _, full in GATED.values() if full} == {WIDE, SMALL_FLOAT}, product
    # no size takes another
    seen = {t: set() for t in KINDS}
    for rows in (1, 30, 200, 1000, 5000, 20000, 100000, 1 << 20):
        for cols in (1, 20, 122, 500, 2000, 9000, 30000):
            for hidden in (1, 40, 64, 300, 1500, 7000, 30000):
                for t in KINDS:
                    if max(rows * cols, rows * hidden) <= 1 << 35:
                        seen[t].update(_tiles(t, (rows, cols, hidden)))
    assert seen[F16] == seen[BF16] == {LARGE, ALONE, MIDDLE, SMALL} and seen[F32] == {WIDE, SMALL_FLOAT, 0}
    lib, tiles = hive_gpu.load_library(), (ctypes.c_int * 3)()
    for bad in ((3, 1, 1, 1, tiles), (0, 0, 1, 1, tiles), (0, 1, 0, 1, tiles), (0, 1 << 21, 1, 1, tiles), (0, 1, 1, 1, None)):
        assert lib.hg_gated_tiles(*bad) == 1, bad


@pytest.mark.gpu
@pytest.mark.parametrize("t,sizes", [(t, s) for s, (_, full) in GATED.items() for t in KINDS if t != F32 or full], ids=str)
def test_gated_in_every_tile(ext, t, sizes):  # noqa: F811
    _check_gated(ext, *_gated(*sizes, t, 5), "silu")
