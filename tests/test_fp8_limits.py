"""Sizes that the E4M3 blocks refuse because no launch holds them.

The C entry points check their arguments on the host, so no GPU is needed and the
addresses are never read."""

import ctypes
import os

import pytest

from mega_moe import _lib

built = pytest.mark.skipif(not os.path.exists(_lib.library_path()), reason="libmegamoe.so not built")
FAKE = ctypes.c_void_p(1 << 20)
TILES = 1 << 22  # of 1024 threads: 2^32 of them


@built
@pytest.mark.parametrize("xt", [0, 1, 2])  # bf16, fp16, fp32
@pytest.mark.parametrize("rows,cols", [(TILES * 128, 1), (TILES * 128 - 127, 128), (TILES * 64, 129), (512 * 128, 8193 * 128)])
def test_blocks_of_rows_and_columns_refuse_what_no_grid_holds(xt, rows, cols):
    """A scale for each row and column: tiles of 1024 threads, fewer than 2^32 threads in all."""
    lib = _lib.load()
    tiles = -(-rows // 128) * -(-cols // 128)
    assert tiles >= TILES and tiles < 1 << 24
    assert lib.mm_quantize_blocks_t(FAKE, cols, xt, None, rows, cols, 1, FAKE, FAKE, FAKE, FAKE, None) == -1
    assert b"too many" in lib.mm_last_error()


@built
def test_square_blocks_refuse_what_no_grid_holds():
    """One scale for 128 x 128: from 2^24 tiles of 256 threads on."""
    lib = _lib.load()
    assert lib.mm_quantize_blocks(FAKE, 128 * 128, 0, 0, 1, 1 << 24, 128 * 128, 128, FAKE, 128 * 128, FAKE, None) == -1
    assert b"too many" in lib.mm_last_error()
    assert lib.mm_quantize_blocks_t(FAKE, 128 * 128, 4, FAKE, 1 << 24, 128 * 128, 128, None, None, FAKE, FAKE, None) == -1
    assert b"too many" in lib.mm_last_error()
