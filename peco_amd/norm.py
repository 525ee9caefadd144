"""Layer norm over the channels of rows on gfx950: forward, backward, and with rows that come out in 8 bits.

``layer_norm`` is the norm of a transformer block, with a weight and a bias for all rows or a modulation of each batch
entry; ``LayerNorm`` is torch's module on it, and ``layer_norm_rows`` quantizes the rows as it makes them, for
``projection.int8_linear``.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _native
from .projection import QuantizedRows, empty_codes, outer_axes

_TYPES = (torch.float16, torch.bfloat16, torch.float32)
_MOST_CHANNELS = 16384
_LONGS = {n: ctypes.c_int64 * n for n in (3, 6, 9)}


def _check(x, weight, bias, eps, around_one, name):
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        raise ValueError(f"{name} expects rows [..., C]")
    dtype, device, shape = x.dtype, x.device, x.shape
    if dtype not in _TYPES:
        raise TypeError(f"{name} supports float16, bfloat16 and float32")
    channels = shape[-1]
    if not 1 <= channels <= _MOST_CHANNELS:
        raise ValueError(f"{name} supports rows of 1 to {_MOST_CHANNELS} channels")
    if not isinstance(eps, (int, float)) or not 0.0 <= eps <= 1e30:
        raise ValueError("eps must be a nonnegative finite number")
    if around_one and weight is None:
        raise ValueError("around_one needs a weight")
    for t in (weight, bias):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or (t.dtype is not dtype and t.dtype is not torch.float32):
            raise TypeError("weight and bias must be tensors of the rows' dtype or float32")
        if t.shape[-1:] != shape[-1:] or (t.dim() != 1 and (t.dim() != 2 or len(shape) < 2 or t.shape[0] != shape[0])):
            raise ValueError("weight and bias must have shape [C], or [B, C] with B the rows' first axis")
        if t.device != device:
            raise ValueError("weight and bias must reside on the device of the rows")
    if not x.is_cuda:
        raise ValueError("peco_amd layer norms run on GPU tensors; CPU tensors are not supported")
    tensors = (x,) if weight is None else (x, weight)
    if not _native.plain_tensors(*(tensors if bias is None else (*tensors, bias))):
        raise RuntimeError(f"{name} takes ordinary tensors (no tracing, transforms or tangents)")
    if x.numel() >= channels << 30:
        raise ValueError(f"{name} supports fewer than 2^30 rows")
    if weight is not None and bias is not None and (weight.dtype != bias.dtype or weight.dim() != bias.dim()):
        _native.retain(x.device, weight, bias)  # (read by what follows)
        weight, bias = weight.float(), bias.float()  # one type, one shape
        if weight.dim() != bias.dim():
            weight, bias = weight.expand(shape[0], channels), bias.expand(shape[0], channels)
    return weight, bias


def _records(x, weight, bias):
    """Whether a gradient of some input is recorded."""
    return torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                        (bias is not None and bias.requires_grad))


def _affine(weight, bias):
    """(weight, bias, elements between two entries' weights, whether they are fp32) as the kernels take them."""
    one = bias if weight is None else weight
    if one is None:
        return None, None, 0, 0
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    return weight, bias, one.shape[1] if one.dim() == 2 else 0, int(one.dtype == torch.float32)


def _channels_adjacent(t):
    return t if t.stride(-1) == 1 else t.contiguous()


def _launch(x, weight, bias, eps, around_one, want_stats):
    """(output, statistics, what a gradient call takes again); the last two None without ``want_stats``."""
    out = torch.empty_like(x)
    if x.numel() == 0:
        return out, None, None
    device, channels, stats, plan = x.device, x.shape[-1], None, None
    with _native.on_device(device):
        _native.require_gfx950(device)
        source, sizes, strides = outer_axes(_channels_adjacent(x))
        target, to = out, strides
        if out.stride() != source.stride():
            _, _, to = outer_axes(target, copy=False)
            if to is None or out.stride(-1) != 1:
                target = torch.empty(x.shape, dtype=x.dtype, device=device)
                _, _, to = outer_axes(target)
        given = weight, bias
        weight, bias, entry, wide = _affine(weight, bias)
        code = _native.dtype_code(x.dtype)
        if want_stats:
            stats = torch.empty((x.numel() // channels, 3), dtype=torch.float32, device=device)
            plan = sizes, channels, entry, wide, code
        address = _native.address
        _native.check(_native.library().peco_layer_norm(
            source.data_ptr(), target.data_ptr(), _LONGS[6](*strides, *to), address(weight), address(bias), entry, wide,
            int(around_one), eps, address(stats), *sizes, channels, code,
            _native.retain(device, x, *given)), "PECO HIP layer norm")
        return out if target is out else out.copy_(target), stats, plan


@functools.lru_cache(maxsize=1024)
def _grad_floats(device_index, *sizes):
    """The workspace of a gradient call; it depends on the sizes and on the device's compute units alone."""
    return _native.library().peco_layer_norm_grad_workspace_size(*sizes)


def _kind(t):
    return None if t is None else (t.shape, t.dtype, t.device)


def _gradients(ctx, grad):
    """Gradients of x, weight and bias, None where none is asked for.

    Few steps: torch's engine calls this on a thread of its own, whose core has to fetch everything that it touches (a
    step costs two to three times what it does on the caller's). The engine has made the forward's device and stream
    the current ones, on which the forward recorded the tensors it saved.
    """
    if not _native.plain_gradient(grad):
        raise RuntimeError("the gradient of layer_norm's output must be an ordinary tensor (no tracing, transforms, "
                           "batches or tangents)")
    x, weight, bias, stats = saved = ctx.saved_tensors
    if tuple(map(_kind, saved)) != ctx.kinds:
        raise RuntimeError("a tensor that layer_norm saved for its gradient has another shape, dtype or device now")
    needs, dense = ctx.needs_input_grad, torch.contiguous_format
    dx = torch.empty_like(x, memory_format=dense) if needs[0] else None
    dweight = torch.empty_like(weight, memory_format=dense) if needs[1] else None
    dbias = torch.empty_like(bias, memory_format=dense) if needs[2] else None
    if ctx.plan is None:  # no rows
        return dx, *(None if t is None else t.zero_() for t in (dweight, dbias)), None, None
    sizes, channels, entry, wide, code = ctx.plan
    source, _, strides = outer_axes(_channels_adjacent(x))  # (hooks of saved tensors may lay out x and stats anew)
    stats = stats.contiguous()
    above, _, by = outer_axes(_channels_adjacent(grad))
    rows = sizes[2] * channels
    workspace, floats, device = None, 0, x.device
    if needs[1] or needs[2]:
        floats = _grad_floats(device.index, *sizes, channels, int(entry > 0))
        workspace = torch.empty(floats, dtype=torch.float32, device=device)
    if weight is not None:
        weight = weight.contiguous()
    address = _native.address
    status = _native.library().peco_layer_norm_grad(
        source.data_ptr(), above.data_ptr(), address(dx), _LONGS[9](*strides, *by, sizes[1] * rows, rows, channels),
        address(weight), 0 if weight is None else entry, wide, ctx.around_one, stats.data_ptr(), address(dweight),
        address(dbias), int(entry > 0), address(workspace), floats, *sizes, channels, code, _native.retain(device, grad))
    if status:
        _native.check(status, "PECO HIP layer norm gradient")
    return dx, dweight, dbias, None, None


_graph_of_gradients = torch.autograd.function.once_differentiable(_gradients)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, around_one):
        out, stats, ctx.plan = _launch(x, weight, bias, eps, around_one, True)
        saved = x, weight, bias, stats
        ctx.save_for_backward(*saved)
        ctx.kinds = tuple(map(_kind, saved))
        ctx.around_one = int(around_one)
        return out

    @staticmethod
    def backward(ctx, grad):
        # (The wrapper costs as much as a launch; without a graph of the gradients it changes nothing.)
        return _graph_of_gradients(ctx, grad) if torch.is_grad_enabled() else _gradients(ctx, grad)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-6, *, around_one: bool = False) -> torch.Tensor:
    """Rows x [..., C] less their mean, over their deviation sqrt(variance + eps), times the weight, plus the bias.

    fp16, bf16 or fp32 rows of 1 to 16384 channels, any strides (rows whose channels are not adjacent are copied
    first); the result has the strides of ``empty_like(x)``. Weight and bias have the rows' dtype or float32 and shape
    [C], or [B, C]: one for each entry of the rows' first axis, as a block's modulation gives them. ``around_one``
    multiplies with 1 + weight. Statistics and arithmetic are fp32, the result is rounded once. A row with an
    infinity or a NaN gives NaN and leaves the others as they are. Rows with deviations past 10^19, whose squares leave
    fp32, are out of its range.

    Differentiable once in x, weight and bias; all sums of the gradients are fp32 in a fixed order, so they repeat bit for
    bit. The gradient of the result must be an ordinary tensor (no batch of gradients, no tangent). A backward pass may be
    captured into a HIP graph while no eager graph of the same leaves is alive (torch's engine would accumulate their
    gradients on that graph's stream and end the process).
    """
    weight, bias = _check(x, weight, bias, eps, around_one, "layer_norm")
    if _records(x, weight, bias):
        if x.dim() > 1 and x.shape[0] > 65535 and any(t is not None and t.dim() == 2 for t in (weight, bias)):
            raise ValueError("gradients support weights of at most 65535 entries")
        return _LayerNorm.apply(x, weight, bias, eps, around_one)
    return _launch(x, weight, bias, eps, around_one, False)[0]


def layer_norm_rows(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                    eps: float = 1e-6, *, around_one: bool = False) -> QuantizedRows:
    """``projection.quantize_rows`` of ``layer_norm``'s rows in one pass, which take their codes from their fp32 values
    (they are not rounded to x's dtype on the way). For inference: it has no gradient."""
    weight, bias = _check(x, weight, bias, eps, around_one, "layer_norm_rows")
    if _records(x, weight, bias):
        raise RuntimeError("layer_norm_rows supports inference only; use torch.no_grad()")
    codes, scales, pitch = empty_codes(x)
    if x.numel():
        device = x.device
        with _native.on_device(device):
            _native.require_gfx950(device)
            source, sizes, strides = outer_axes(_channels_adjacent(x))
            given = weight, bias
            weight, bias, entry, wide = _affine(weight, bias)
            _native.check(_native.library().peco_layer_norm_rows(
                source.data_ptr(), _LONGS[3](*strides), _native.address(weight), _native.address(bias), entry, wide,
                int(around_one), eps, codes.data_ptr(), pitch, scales.data_ptr(), *sizes, x.shape[-1],
                _native.dtype_code(x.dtype), _native.retain(device, x, *given)), "PECO HIP layer norm")
    return QuantizedRows(codes, scales)


class LayerNorm(torch.nn.LayerNorm):
    """``torch.nn.LayerNorm`` over the last axis by ``layer_norm``; its results have the rows' dtype, under autocast too."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        if len(self.normalized_shape) != 1:
            raise ValueError("LayerNorm normalises over the last axis alone")

    def forward(self, x):
        if x.shape[-1:] != self.normalized_shape:
            raise ValueError(f"Expected rows of {self.normalized_shape[0]} channels, got {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)
