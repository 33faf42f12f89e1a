"""The sizes of the E4M3 products' GPU tests reach every tile that there is.

Tiles are chosen by measured costs; where those are measured again, a tile that no
tested size takes any more is named here."""

import pytest

from tests import _fp8_tiles as T
from tests.test_gpu_fp8_tiles import SIZES

# rows, channels, K of products in the other files: tiles of up to 64 rows
SMALL = [(64, 512, 1024), (255, 384, 4096), (33, 129, 257), (1021, 1030, 1153), (1000, 1900, 2100), (100, 1000, 1000),
         (65, 300, 131)]


@pytest.mark.parametrize("size", SIZES)
def test_sizes_take_the_tiles_they_are_for(size):
    m, n, k, _, _, half, full = size
    assert T.tile(m, n, k, False) == half and T.tile(m, n, k, True) == full


@pytest.mark.parametrize("wide,table", [(False, "kTileCosts"), (True, "kWideCosts")])
def test_every_tile_is_tested(wide, table):
    tiles = {(bm, bn) for bm, bn, *_ in T.costs(table)}
    assert len(tiles) >= 4
    assert {T.tile(m, n, k, wide) for m, n, k, *_ in SIZES + SMALL} == tiles
