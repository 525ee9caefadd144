"""C entries of the 8-bit product: results that no launch of the product's kernel holds are refused before the rows are
quantized and before the workspace is looked at (no GPU is reached)."""
import ctypes

import pytest

from peco_amd import _native

SOME, NULL = ctypes.c_void_p(4096), ctypes.c_void_p(0)  # (refused before it is read)
SMALL, SHAPE = 20001, 20002


def _product_rows(rows, outputs, x_dtype):
    return _native.library().peco_int8_linear_rows(SOME, (ctypes.c_int64 * 3)(64, 64, 64), rows, 1, 1, x_dtype, SOME, 64, SOME,
                                                   NULL, 0, SOME, NULL, 0, 64, outputs, 1, NULL)


# Few rows: 16 outputs a workgroup of 512 lanes. 33 to 64 rows of that many outputs: middle tiles, 128 a workgroup of 512.
@pytest.mark.parametrize("rows,outputs", [(1, 1 << 27), (16, (1 << 27) + 5), (17, 1 << 27), (32, (1 << 30) - 1),
                                          (33, (1 << 30) - 1), (128, (1 << 30) - 127), (1 << 29, 1 << 29)])
def test_products_that_no_launch_holds(rows, outputs):
    assert _product_rows(rows, outputs, 2) == SHAPE
    assert _native.library().peco_int8_linear(SOME, 64, SOME, SOME, 64, SOME, NULL, 0, SOME, rows, 64, outputs, 1, NULL) == SHAPE


@pytest.mark.parametrize("rows,outputs", [(16, (1 << 27) - 16), (32, (1 << 27) - 16), (33, (1 << 30) - 129)])
def test_the_largest_that_one_holds_come_to_the_workspace(rows, outputs):
    assert _product_rows(rows, outputs, 2) == SMALL
