"""Room for the column sums of layer norm's backward pass, without a GPU (148 SMs are assumed then): two rows of
sums for each block that a plan can launch, which is far less than the input for wide rows."""
import pytest

from conftest import pkg_module


def room(rows, cols):
    return pkg_module("_lib").load().f16_layer_norm_scratch_floats(rows, cols)


@pytest.mark.parametrize("rows,cols", [(1000, 1_000_000), (2000, 1_000_000), (6700, 20001), (4096, 16384), (300, 2 ** 29)])
def test_wide_rows_take_a_few_slices(rows, cols):
    """Tiles of 256 threads x 8 values at most; slices so that four blocks an SM are busy."""
    tiles = -(-cols // (256 * 8))
    slices = min(rows, -(-4 * 148 // tiles))
    assert 2 * cols <= room(rows, cols) <= 2 * cols * slices


@pytest.mark.parametrize("rows,cols,blocks", [(16384, 4096, 296), (524288, 512, 1184), (524288, 256, 296), (100003, 215, 296),
                                              (16384, 8192, 148), (50000, 4097, 592)])
def test_rows_in_registers_take_what_their_blocks_write(rows, cols, blocks):
    """16 warps an SM: two blocks of 256 threads, one of 512, and eight of 64 where 512 columns are not aligned for
    16-byte loads (8 values a thread); at 4,097 16-bit columns rows are read again (592 slices over 3 or 17 tiles)."""
    assert room(rows, cols) <= 2 * cols * blocks


def test_few_rows():
    for cols in (1, 8, 215, 4096, 20001):
        for rows in (1, 2, 3):
            assert 2 * cols <= room(rows, cols) <= 2 * cols * rows
