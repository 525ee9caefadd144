"""Calls whose launches would have 2^32 lanes or more are refused before any of their launches (no GPU is reached)."""
import ctypes

import pytest
import torch

from peco_amd import _native
from peco_amd.rotary import RotaryAxes, plan_arguments

SOME, NULL = ctypes.c_void_p(4096), ctypes.c_void_p(0)  # (refused before it is read)
REFUSED = 20002


def _strides(n):
    return (ctypes.c_int64 * n)(*[64] * n)


@pytest.mark.parametrize("batch,queries", [((1 << 21) + 1, 1), (1 << 14, 128 * 129)])
@pytest.mark.parametrize("dim,dtype", [(64, 0), (128, 1)])
def test_window(batch, queries, dim, dtype):
    """8 heads: past 2^24 workgroups of 256 lanes, a row tile each."""
    sizes = (batch, 8, 8, queries, queries, 10, 0, 0)
    lib = _native.library()
    floats = lib.peco_window_attention_workspace_size(*sizes, dim)
    assert lib.peco_window_attention(SOME, SOME, SOME, SOME, _strides(12), NULL, NULL, NULL, NULL, SOME, floats, *sizes, 0.125,
                                     dim, dtype, NULL) == REFUSED
    floats = lib.peco_window_attention_grad_workspace_size(*sizes, dim, dtype)
    assert lib.peco_window_attention_grad(SOME, SOME, SOME, SOME, SOME, SOME, SOME, SOME, _strides(24), NULL, SOME, SOME, SOME,
                                          SOME, floats, *sizes, 0.125, dim, dtype, NULL) == REFUSED


def test_paged():
    lib = _native.library()
    sizes, page, width = ((1 << 21) + 1, 24, 8, (1 << 21) + 1), 16, 4
    floats = lib.peco_paged_attention_workspace_size(*sizes, width, page, -1, 0, 64)
    assert lib.peco_paged_attention(SOME, SOME, SOME, SOME, _strides(10), SOME, width, SOME, SOME, 0, SOME, floats, *sizes, 9,
                                    page, width, -1, 0, 0.125, 64, 1, NULL) == REFUSED


def test_append():
    lib = _native.library()
    plan = plan_arguments(RotaryAxes((16, 24, 24)), torch.zeros(3, 3, dtype=torch.int32))
    tokens = (1 << 28) + 1  # 16 lanes a token
    assert lib.peco_append_pages(SOME, SOME, SOME, SOME, _strides(10), SOME, 4, SOME, SOME, *plan, 1, 2, tokens, 9, 16, 4, 128,
                                 1, NULL) == REFUSED
