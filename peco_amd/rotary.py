"""Rotary positions with several axes (time, height, width, ...) on gfx950.

``RotaryAxes`` says how the channels of a row are divided over the axes and how fast each pair of channels
turns; ``rotary_axes`` turns rows by their positions, computing the angles in the kernel (in 64 bits up to the
fraction of a turn), with a gradient. ``PecoAttention.__call__`` takes a ``RotaryPositions`` as its
``image_rotary_emb`` in place of (cos, sin) tables, and ``paged.append_pages`` turns keys on their way into a
cache with one.

With ``theta=256`` and axes (16, 56, 56) over 128 channels the angles are those of HunyuanVideo's tables.
"""
from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass

import torch

from . import _native

_LAYOUTS = ("interleaved", "halves")
_POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
_MAX_AXES, _MAX_PAIRS = 4, 128


@dataclass(frozen=True)
class RotaryAxes:
    """How rows turn: ``dims[a]`` channels of a row turn with axis a (in order; channels behind the last axis
    stay as they are), pair i of an axis by ``position * theta ** (-2 i / dims[a])``.

    ``layout`` "interleaved" pairs adjacent channels (2 i, 2 i + 1), "halves" channels (i, i + sum(dims) / 2).
    ``shared`` takes one ladder of frequencies over all pairs, ``theta ** (-2 i / sum(dims))`` with i counted
    through the axes, in place of one for each axis.
    """

    dims: tuple
    theta: float = 10000.0
    layout: str = "interleaved"
    shared: bool = False

    def __post_init__(self):
        dims = tuple(self.dims)
        if not 1 <= len(dims) <= _MAX_AXES or any(not isinstance(d, int) or d < 2 or d % 2 for d in dims):
            raise ValueError(f"dims must be 1 to {_MAX_AXES} positive even integers")
        if sum(dims) > 2 * _MAX_PAIRS:
            raise ValueError(f"the axes may turn at most {2 * _MAX_PAIRS} channels")
        if not isinstance(self.theta, (int, float)) or not math.isfinite(self.theta) or self.theta <= 0:
            raise ValueError("theta must be a positive finite number")
        if self.layout not in _LAYOUTS:
            raise ValueError(f"layout must be one of {_LAYOUTS}")
        if self.layout == "halves" and sum(dims) % 16:
            raise ValueError("layout 'halves' needs the axes' channels to sum to a multiple of 16")
        object.__setattr__(self, "dims", dims)

    @staticmethod
    def grid(frames, rows, columns, *, first_frame=0, device=None):
        """Positions int32 [3, frames * rows * columns] of a clip's tokens in (frame, row, column) order."""
        axes = torch.meshgrid(torch.arange(first_frame, first_frame + frames, dtype=torch.int32),
                              torch.arange(rows, dtype=torch.int32), torch.arange(columns, dtype=torch.int32),
                              indexing="ij")
        return torch.stack([a.reshape(-1) for a in axes]).to(device)


@dataclass(frozen=True, eq=False)
class RotaryPositions:
    """Rows' positions (as ``rotary_axes`` takes them) together with the axes they turn with."""

    axes: RotaryAxes
    positions: torch.Tensor


@functools.lru_cache(maxsize=64)
def _plan(axes: RotaryAxes):
    """(turns per unit of position of each pair, pairs of each axis) as host arrays of the C-ABI."""
    total = sum(axes.dims)
    turns, first = [], 0
    for d in axes.dims:
        for i in range(d // 2):
            step = 2 * (first + i) / total if axes.shared else 2 * i / d
            turns.append(float(axes.theta) ** -step / (2 * math.pi))
        first += d // 2
    pairs = [d // 2 for d in axes.dims]
    return (ctypes.c_double * len(turns))(*turns), (ctypes.c_int * len(pairs))(*pairs)


def plan_arguments(axes, positions, inverse=False):
    """The plan's arguments of the C-ABI entries, for positions that ``check_positions`` returned."""
    turns, pairs = _plan(axes)
    batch = positions.stride(0) if positions.dim() == 3 and positions.shape[0] > 1 else 0
    return (positions.data_ptr(), _POSITION_TYPES[positions.dtype], batch, positions.stride(-2), turns, pairs,
            len(axes.dims), int(axes.layout == "halves"), int(inverse))


def check_positions(axes, positions, batch, rows, dim, device):
    """Positions [A, rows] or [batch, A, rows] that the kernels can read (rows adjacent), or an error."""
    if not isinstance(axes, RotaryAxes):
        raise TypeError("axes must be a RotaryAxes")
    if sum(axes.dims) > dim:
        raise ValueError("the axes turn more channels than a row has")
    if not isinstance(positions, torch.Tensor) or positions.dtype not in _POSITION_TYPES:
        raise TypeError("positions must be an int32, int64 or float32 tensor")
    shape = (len(axes.dims), rows)
    if positions.shape != shape and positions.shape != (batch, *shape):
        raise ValueError(f"positions must have shape [{len(axes.dims)}, {rows}] or [{batch}, {len(axes.dims)}, {rows}]")
    if positions.device != device:
        raise ValueError("positions must reside on the device of the rows")
    if not _native.plain_tensors(positions):
        raise RuntimeError("rotary positions must be ordinary tensors (no tracing, transforms or tangents)")
    if positions.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("positions have no gradient")
    return positions if positions.stride(-1) == 1 else positions.contiguous()


def _rows16(x):
    """x with adjacent channels and every row of every head on 16 bytes (a copy when it is laid out otherwise)."""
    b, h, r, inner = x.stride()
    if inner == 1 and x.data_ptr() % 16 == 0 and (b | h | r) * x.element_size() % 16 == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _launch(x, positions, axes, inverse):
    out = torch.empty_like(x)
    if x.numel() == 0:
        return out
    batch, heads, rows, dim = x.shape
    device = x.device
    with _native.on_device(device):
        _native.require_gfx950(device)
        source, target = _rows16(x), out
        if _rows16(target) is not target:
            target = torch.empty(x.shape, dtype=x.dtype, device=device)
        status = _native.library().peco_rotary_axes(
            source.data_ptr(), *source.stride()[:3], target.data_ptr(), *target.stride()[:3],
            *plan_arguments(axes, positions, inverse), batch, heads, rows, dim, _native.dtype_code(x.dtype),
            _native.retain(device, source, positions))
        _native.check(status, "PECO HIP rotary positions")
        return out if target is out else out.copy_(target)


class _RotaryAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, axes):
        ctx.save_for_backward(positions)
        ctx.axes = axes
        return _launch(x, positions, axes, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        if not _native.plain_gradient(grad):
            raise RuntimeError("the gradient of rotary_axes' output must be an ordinary tensor (no tracing, transforms, "
                               "batches or tangents)")
        return _launch(grad, ctx.saved_tensors[0], ctx.axes, True), None, None


def rotary_axes(x: torch.Tensor, positions: torch.Tensor, axes: RotaryAxes) -> torch.Tensor:
    """Rows x [B,H,S,D] turned by their positions (int32, int64 or float32 [A,S] or [B,A,S], A the axes).

    fp16, bf16 or fp32 rows, D a multiple of 8 up to 512, any strides (rows that are not laid out on 16 bytes
    with adjacent channels are copied first); the result has the strides of ``empty_like(x)``. Differentiable
    once in x: its gradient is turned back (a backward pass may be captured into a HIP graph while no eager graph
    of the same leaf is alive, as with any torch operation). Rows are turned in fp32 and rounded once.
    """
    if not isinstance(x, torch.Tensor) or x.dim() != 4:
        raise ValueError("rotary_axes expects rows [B,H,S,D]")
    if x.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError("rotary_axes supports float16, bfloat16 and float32")
    if x.shape[3] % 8 or not 8 <= x.shape[3] <= 512:
        raise ValueError("rotary_axes supports row lengths that are multiples of 8 up to 512")
    positions = check_positions(axes, positions, x.shape[0], x.shape[2], x.shape[3], x.device)
    if not x.is_cuda:
        raise ValueError("peco_amd rotary positions run on GPU tensors; CPU tensors are not supported")
    if not _native.plain_tensors(x):
        raise RuntimeError("rotary_axes takes ordinary tensors (no tracing, transforms or tangents)")
    if torch.is_grad_enabled() and x.requires_grad:
        return _RotaryAxes.apply(x, positions, axes)
    return _launch(x, positions, axes, False)
