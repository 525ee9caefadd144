"""C entries of the norms and 8-bit projections: bad arguments are refused before any launch (no GPU is reached)."""
import ctypes

import pytest

from peco_amd import _native

SOME, NULL = ctypes.c_void_p(4096), ctypes.c_void_p(0)  # (refused before it is read)
INVALID, SMALL, SHAPE, DTYPE = 1, 20001, 20002, 20003


def _strides(n):
    return (ctypes.c_int64 * n)(*[64] * n)


def _norm(x=SOME, out=SOME, strides=_strides(6), entry=0, sizes=(2, 3, 5), channels=64, dtype=1):
    return _native.library().peco_layer_norm(x, out, strides, SOME, SOME, entry, 0, 0, 1e-6, NULL, *sizes, channels, dtype, NULL)


def _rows(entry_point, x=SOME, codes=SOME, pitch=64, scales=SOME, sizes=(2, 3, 5), channels=64, dtype=1):
    lib = _native.library()
    if entry_point == "norm":
        return lib.peco_layer_norm_rows(x, _strides(3), SOME, SOME, 0, 0, 0, 1e-6, codes, pitch, scales, *sizes, channels,
                                        dtype, NULL)
    return lib.peco_quantize_rows(x, _strides(3), codes, pitch, scales, *sizes, channels, dtype, NULL)


def _grad(x=SOME, dx=SOME, entry=0, dweight=SOME, dbias=SOME, per_entry=0, floats=1 << 30, workspace=SOME, sizes=(2, 3, 5),
          channels=64, dtype=1):
    return _native.library().peco_layer_norm_grad(x, SOME, dx, _strides(9), SOME, entry, 0, 0, SOME, dweight, dbias, per_entry,
                                                  workspace, floats, *sizes, channels, dtype, NULL)


def _product(codes=SOME, pitch=64, weight=SOME, weight_pitch=64, out=SOME, rows=30, channels=64, outputs=40, dtype=1):
    return _native.library().peco_int8_linear(codes, pitch, SOME, weight, weight_pitch, SOME, NULL, 0, out, rows, channels,
                                              outputs, dtype, NULL)


def _product_rows(x=SOME, sizes=(2, 30, 50), x_dtype=1, weight_pitch=64, workspace=SOME, size=1 << 40, channels=64, outputs=40,
                  dtype=1):
    return _native.library().peco_int8_linear_rows(x, _strides(3), *sizes, x_dtype, SOME, weight_pitch, SOME, NULL, 0, SOME,
                                                   workspace, size, channels, outputs, dtype, NULL)


def test_layer_norm():
    for change, status in ((dict(x=NULL), INVALID), (dict(out=NULL), INVALID), (dict(strides=None), INVALID),
                           (dict(entry=-1), INVALID), (dict(sizes=(0, 3, 5)), INVALID), (dict(channels=0), INVALID),
                           (dict(channels=16385), SHAPE), (dict(sizes=(1 << 10, 1 << 10, 1 << 10)), SHAPE),
                           (dict(sizes=(1 << 16, 1 << 16, 1)), SHAPE), (dict(dtype=3), DTYPE)):
        assert _norm(**change) == status, change


@pytest.mark.parametrize("entry_point", ["norm", "rows"])
def test_rows(entry_point):
    for change, status in ((dict(x=NULL), INVALID), (dict(codes=NULL), INVALID), (dict(scales=NULL), INVALID),
                           (dict(pitch=63), INVALID), (dict(pitch=48), INVALID), (dict(pitch=72), INVALID),
                           (dict(codes=ctypes.c_void_p(4100)), INVALID), (dict(channels=16385, pitch=1 << 20), SHAPE),
                           (dict(dtype=-1), DTYPE)):
        assert _rows(entry_point, **change) == status, change


def test_gradients():
    lib = _native.library()
    floats = lib.peco_layer_norm_grad_workspace_size(2, 3, 5, 64, 1)
    assert floats >= 2 * 2 * 64
    assert lib.peco_layer_norm_grad_workspace_size(2, 3, 5, 16385, 0) == 0
    assert lib.peco_layer_norm_grad_workspace_size(65536, 1, 1, 64, 1) == 0
    for change, status in ((dict(x=NULL), INVALID), (dict(entry=64), INVALID), (dict(entry=-64, per_entry=1), INVALID),
                           (dict(dx=NULL, dweight=NULL, dbias=NULL), INVALID), (dict(sizes=(2, 0, 5)), INVALID),
                           (dict(channels=16385), SHAPE), (dict(sizes=(65536, 1, 1), per_entry=1, entry=64), SHAPE),
                           (dict(dtype=7), DTYPE), (dict(workspace=NULL), SMALL),
                           (dict(per_entry=1, entry=64, floats=floats - 1), SMALL)):
        assert _grad(**change) == status, change


def test_product():
    for change, status in ((dict(codes=NULL), INVALID), (dict(weight=NULL), INVALID), (dict(out=NULL), INVALID),
                           (dict(pitch=65), INVALID), (dict(weight_pitch=-16), INVALID), (dict(weight_pitch=40), INVALID),
                           (dict(out=ctypes.c_void_p(4104)), INVALID), (dict(rows=0), INVALID), (dict(outputs=0), INVALID),
                           (dict(channels=1 << 17), SHAPE), (dict(pitch=(1 << 22) + 16), SHAPE),
                           (dict(rows=1 << 29, outputs=1 << 29), SHAPE), (dict(rows=1 << 30), SHAPE), (dict(dtype=3), DTYPE)):
        assert _product(**change) == status, change


def test_product_of_rows():
    lib = _native.library()
    assert lib.peco_int8_linear_rows_workspace_size(1, 2048, 1, 1) == 0  # quantized by the product's launch
    assert lib.peco_int8_linear_rows_workspace_size(1, 2048, 2, 1) == 2048 + 4
    assert lib.peco_int8_linear_rows_workspace_size(3000, 70, 1, 1) == 3000 * (80 + 4)
    assert lib.peco_int8_linear_rows_workspace_size(3000, 1000, 1, 1) == 3000 * (1024 + 4)
    assert lib.peco_int8_linear_rows_workspace_size(3000, 16385, 1, 1) == 0
    for change, status in ((dict(x=NULL), INVALID), (dict(sizes=(0, 1, 1)), INVALID), (dict(x_dtype=3), DTYPE),
                           (dict(dtype=3), DTYPE), (dict(channels=16385, weight_pitch=1 << 20), SHAPE),
                           (dict(sizes=(1 << 10, 1 << 10, 1 << 10)), SHAPE), (dict(weight_pitch=72), INVALID),
                           (dict(sizes=(1, 1 << 14, 1 << 15), outputs=1 << 29), SHAPE), (dict(workspace=NULL), SMALL),
                           (dict(size=3000 * (64 + 4) - 1), SMALL), (dict(workspace=ctypes.c_void_p(4104)), INVALID)):
        assert _product_rows(**change) == status, change
