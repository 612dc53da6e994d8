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
from test_gpu_network_ops import (BF16, F16, F32, HALF_ULP, U, _check_gated, _gated, _iteration, _muon_reference,  # noqa: F401
                                  _randn, ext)

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

# (matrices, rows, columns): the tiles of A and P, and of P X
TEAMS, MIDDLE_PARTS, LARGE_PARTS, SMALL_PARTS = 106406441, 12812822, 25625621, 6406442
MATRICES = {
    (1, 65, 65): (TEAMS, TEAMS),
    (3, 1100, 260): (TEAMS, SMALL_PARTS),
    (4, 1040, 2056): (SMALL_PARTS, MIDDLE_PARTS),
    (5, 1040, 2056): (MIDDLE_PARTS, LARGE_PARTS),
    (12, 650, 1100): (MIDDLE_PARTS, MIDDLE_PARTS),
    (6, 2056, 1040): (MIDDLE_PARTS, LARGE_PARTS),
    (40, 130, 3001): (TEAMS, LARGE_PARTS),
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


def _matrix_tiles(*sizes):
    tiles = (ctypes.c_int * 2)()
    assert hive_gpu.load_library().hg_orthogonalize_tiles(*sizes, tiles) == 0
    return tuple(tiles)


@pytest.mark.skipif(not os.path.exists(hive_gpu.LIB_PATH), reason="libhive_gpu.so not built")
def test_the_matrices_below_take_every_tile():
    for sizes, tiles in MATRICES.items():
        assert _matrix_tiles(*sizes) == tiles, sizes
    assert {a for a, _ in MATRICES.values()} == {TEAMS, MIDDLE_PARTS, SMALL_PARTS}
    assert {x for _, x in MATRICES.values()} == {TEAMS, MIDDLE_PARTS, SMALL_PARTS, LARGE_PARTS}
    assert _matrix_tiles(1, 64, 256) == _matrix_tiles(500, 256, 64) == (0, 0) != _matrix_tiles(1, 64, 257)
    seen = [set(), set()]
    for count in (1, 3, 10, 40, 200, 3000):
        for rows in (1, 64, 65, 300, 1000, 4000, 9000):
            for cols in (1, 64, 65, 300, 1000, 4000, 9000):
                if count * (rows // 64 + 1) * (cols // 64 + 1) <= 2049 ** 2:
                    for s, t in zip(seen, _matrix_tiles(count, rows, cols)):
                        s.add(t)
    assert seen == [{0, TEAMS, MIDDLE_PARTS, SMALL_PARTS}, {0, TEAMS, MIDDLE_PARTS, SMALL_PARTS, LARGE_PARTS}]
    lib, tiles = hive_gpu.load_library(), (ctypes.c_int * 2)()
    for bad in ((0, 1, 1, tiles), (1, 0, 1, tiles), (1, 1, 1 << 18, tiles), (1 << 17, 1, 1, tiles), (1, 1, 1, None)):
        assert lib.hg_orthogonalize_tiles(*bad) == 1, bad


def _two_in_turn(shape, seed):
    """A batch of two different matrices in turn: the others of a kind have to be the same bits."""
    two = _randn((min(2, shape[0]), *shape[1:]), seed, 0.03)
    return two, two.repeat((shape[0] + 1) // 2, 1, 1)[:shape[0]].contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", MATRICES, ids=str)
def test_orthogonalize_in_every_tile(ext, sizes):  # noqa: F811
    """To the rounding of 22 bits, and no worse than eight times float32 products' error."""
    two, u = _two_in_turn(sizes, 4)
    got = ext.orthogonalize(u)
    for i in range(2, sizes[0]):
        assert torch.equal(got[i], got[i % 2]), i
    for g, one in zip(got, two):
        want, error = _iteration(one)
        plain, _ = _iteration(one, kind=F32)
        off = float((g.double() - want).norm())
        assert off <= error + U * float(want.norm()) and off <= 8 * float((plain.double() - want).norm())


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16], ids=str)
@pytest.mark.parametrize("sizes", [s for s in MATRICES if LARGE_PARTS in MATRICES[s]], ids=str)
def test_a_step_in_the_largest_tiles(ext, sizes, t):  # noqa: F811
    two, grads = _two_in_turn(sizes, 6)
    params = [_randn(sizes[1:], i % 2, 0.1, t) for i in range(min(sizes[0], 24))]
    before = [p.clone() for p in params[:2]]
    ext.prepare_muon(params).step(list(grads[:len(params)]), lr=0.05, weight_decay=0.1)
    for i in range(2, len(params)):
        assert torch.equal(params[i], params[i % 2]), i
    for p, b, g in zip(params, before, two):
        want, _, error = _muon_reference(b, g, torch.zeros_like(g), 0.05, 0.95, True, 0.1, "spectral")
        off = float((p.double() - want).norm())
        assert off <= error * 1.1 + (HALF_ULP[t] + 4 * U) * float(want.norm()) + 4 * U * 0.05 * float(want.norm() + 8), (off, error)
