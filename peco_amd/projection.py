"""Projections in 8 bits on gfx950: rows quantized with a scale each, times a weight with a scale an output channel.

``quantize_rows`` makes the codes, ``int8_linear`` the product, ``Int8Linear`` is a layer of it in place of
``torch.nn.Linear`` (``model.quantize_projections`` puts it into every attention block of a transformer).

A row's codes are ``rint(x * (127 * (1 / a)))`` with a its largest magnitude, and its scale is ``a * (1 / 127)``, each
operation in fp32, halves to even (for 16-bit rows these are the nearest codes to ``127 x / a``). A row whose largest
magnitude is below 127 * 2^-126 counts as 0. A row with an infinity or a NaN has codes 0 and a NaN as its scale, so its
products are NaN, and no others.
"""
from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass

import torch

from . import _native

_TYPES = (torch.float16, torch.bfloat16, torch.float32)
_MOST_CHANNELS = 16384          # of a row that is quantized
_MOST_PRODUCT = (1 << 17) - 1   # of a product: its sums stay in 32 bits
_LONG3 = ctypes.c_int64 * 3


def outer_axes(t, copy=True):
    """(t, sizes, strides) of the axes of t [..., C] before its channels as three; t is copied where more than three
    axes do not fold into that many (``copy``: else strides None)."""
    n = t.dim() - 1
    shape, stride = t.shape, t.stride()
    if n == 2:
        return t, (shape[0], 1, shape[1]), (stride[0], 0, stride[1])
    if n == 1:
        return t, (shape[0], 1, 1), (stride[0], 0, 0)
    if n == 3:
        return t, tuple(shape[:3]), tuple(stride[:3])
    if n == 0:
        return t, (1, 1, 1), (0, 0, 0)
    middle = shape[1:n - 1].numel()
    try:
        folded = t.view(shape[0], middle, shape[n - 1], shape[n])
    except RuntimeError:
        if not copy:
            return t, None, None
        t = t.contiguous()
        folded = t.view(shape[0], middle, shape[n - 1], shape[n])
    return t, tuple(folded.shape[:3]), tuple(folded.stride()[:3])


def empty_codes(x):
    """Codes like x [..., K] in rows of whole 16 bytes (whole lines for long rows), scales [...], and the rows' distance
    in bytes."""
    *outer, channels = x.shape
    step = 16 if channels < 512 else 128
    pitch = -(-channels // step) * step
    codes = torch.empty((*outer, pitch), dtype=torch.int8, device=x.device)
    return codes if pitch == channels else codes.narrow(-1, 0, channels), \
        torch.empty(outer, dtype=torch.float32, device=x.device), pitch


@dataclass(frozen=True, eq=False)
class QuantizedRows:
    """Rows in 8 bits: ``codes`` int8 [..., K], any strides, and ``scales`` fp32 [...], a row's value being code * scale.

    Rows whose codes start on 16 bytes and lie a fixed distance apart are used in place, others are copied by each call.
    """

    codes: torch.Tensor
    scales: torch.Tensor

    def __post_init__(self):
        if not isinstance(self.codes, torch.Tensor) or not isinstance(self.scales, torch.Tensor):
            raise TypeError("codes and scales must be tensors")
        if self.codes.dtype != torch.int8 or self.scales.dtype != torch.float32:
            raise TypeError("codes must be int8 and scales float32")
        if self.codes.dim() < 1 or self.codes.shape[:-1] != self.scales.shape:
            raise ValueError("codes must have shape [..., K] and scales the same without K")
        if self.codes.device != self.scales.device:
            raise ValueError("codes and scales must reside on the same device")

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        return (self.codes.float() * self.scales[..., None]).to(dtype)


def _check_rows(x, name):
    if x.dim() < 1 or not 1 <= x.shape[-1] <= _MOST_CHANNELS:
        raise ValueError(f"{name} expects rows [..., K] of 1 to {_MOST_CHANNELS} channels")
    if x.dtype not in _TYPES:
        raise TypeError(f"{name} supports float16, bfloat16 and float32")
    if not x.is_cuda:
        raise ValueError("peco_amd projections run on GPU tensors; CPU tensors are not supported")
    if not _native.plain_tensors(x):
        raise RuntimeError(f"{name} takes ordinary tensors (no tracing, transforms or tangents)")
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError(f"{name} supports inference only; use torch.no_grad()")
    if x.numel() // x.shape[-1] >= 1 << 30:
        raise ValueError(f"{name} supports fewer than 2^30 rows")


def quantize_rows(x: torch.Tensor) -> QuantizedRows:
    """Rows x [..., K] (fp16, bf16 or fp32, 1 to 16384 channels, any strides) in 8 bits with a scale each."""
    if not isinstance(x, torch.Tensor):
        raise TypeError("quantize_rows expects a tensor")
    _check_rows(x, "quantize_rows")
    codes, scales, pitch = empty_codes(x)
    if x.numel():
        device = x.device
        with _native.on_device(device):
            _native.require_gfx950(device)
            source, sizes, strides = outer_axes(x if x.stride(-1) == 1 else x.contiguous())
            _native.check(_native.library().peco_quantize_rows(
                source.data_ptr(), _LONG3(*strides), codes.data_ptr(), pitch, scales.data_ptr(), *sizes, x.shape[-1],
                _native.dtype_code(x.dtype), _native.retain(device, x)), "PECO HIP row quantization")
    return QuantizedRows(codes, scales)


def _code_rows(codes):
    """(codes, bytes between rows) as the kernels take them: every row on 16 bytes, a fixed distance apart."""
    stride, shape = codes.stride(), codes.shape
    if stride[-1] == 1 and codes.data_ptr() % 16 == 0:
        if len(shape) == 2 and stride[0] % 16 == 0 and stride[0] <= 1 << 22:
            return codes, stride[0]
        pitch, rows = 0, 1
        for n, s in zip(reversed(shape[:-1]), reversed(stride[:-1])):
            if n == 1:
                continue
            if rows == 1:
                pitch = s
            elif s != rows * pitch:
                pitch = -1
                break
            rows *= n
        if pitch >= 0 and pitch % 16 == 0 and pitch <= 1 << 22:
            return codes, pitch
    kept, _, pitch = empty_codes(codes)
    return kept.copy_(codes), pitch


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(*sizes):
    return _native.library().peco_int8_linear_rows_workspace_size(*sizes)


def int8_linear(x, weight: QuantizedRows, bias: torch.Tensor | None = None, *,
                dtype: torch.dtype | None = None) -> torch.Tensor:
    """x [..., K] times the transpose of ``weight`` [N, K] in 8-bit integers, plus ``bias`` [N]: [..., N].

    x is a tensor (fp16, bf16 or fp32, up to 16384 channels), whose rows are quantized as ``quantize_rows`` does, or
    ``QuantizedRows`` (K below 2^17). The sums over K are exact integers; scales and bias (of the result's dtype or
    float32) are applied in fp32, the row's scale first (the sum times it has to be a number of fp32), and the result is
    rounded once, to ``dtype`` (default: x's, bfloat16 for QuantizedRows). N is below 2^30, for up to 32 rows below 2^27.
    For inference: it has no gradient. Weight rows that do not start on 16 bytes a fixed distance apart are copied by each
    call (``quantize_rows`` lays them out so).
    """
    if not isinstance(weight, QuantizedRows):
        raise TypeError("weight must be QuantizedRows")
    quantized = isinstance(x, QuantizedRows)
    if not quantized and not isinstance(x, torch.Tensor):
        raise TypeError("x must be a tensor or QuantizedRows")
    rows = x.codes if quantized else x
    if weight.codes.dim() != 2 or min(weight.codes.shape) < 1 or rows.dim() < 1 or rows.shape[-1] != weight.codes.shape[1]:
        raise ValueError("Expected x [..., K] and a weight [N, K] that is not empty")
    outputs, channels = weight.codes.shape
    if dtype is None:
        dtype = torch.bfloat16 if quantized else x.dtype
    if dtype not in _TYPES:
        raise TypeError("int8_linear gives float16, bfloat16 or float32")
    device = rows.device
    tensors = [rows, weight.codes, weight.scales]
    if quantized:
        tensors.append(x.scales)
    if bias is not None:
        if not isinstance(bias, torch.Tensor) or bias.dtype not in (dtype, torch.float32):
            raise TypeError("bias must be a tensor of the result's dtype or float32")
        if bias.shape != (outputs,):
            raise ValueError("bias must have shape [N]")
        tensors.append(bias)
    recording = torch.is_grad_enabled()
    for t in tensors:
        if not t.is_cuda or t.device != device:
            raise ValueError("All int8_linear inputs must reside on the same GPU device")
        if recording and t.requires_grad:
            raise RuntimeError("int8_linear supports inference only; use torch.no_grad()")
    if not _native.plain_tensors(*tensors):
        raise RuntimeError("int8_linear takes ordinary tensors (no tracing, transforms or tangents)")
    if quantized:
        if channels > _MOST_PRODUCT:
            raise ValueError(f"int8_linear supports at most {_MOST_PRODUCT} channels")
        if rows.numel() // channels >= 1 << 30:
            raise ValueError("int8_linear supports fewer than 2^30 rows")
    elif channels > _MOST_CHANNELS or rows.numel() // channels >= 1 << 30 or x.dtype not in _TYPES:
        _check_rows(x, "int8_linear")
    if outputs >= 1 << 30:
        raise ValueError("int8_linear supports fewer than 2^30 outputs")
    count = rows.numel() // channels
    if 1 <= count <= 32 and outputs >= 1 << 27:  # (16 a workgroup of 512 lanes, 2^32 lanes a launch)
        raise ValueError("int8_linear supports fewer than 2^27 outputs of up to 32 rows")
    out = torch.empty((*rows.shape[:-1], outputs), dtype=dtype, device=device)
    if count == 0:
        return out
    with _native.on_device(device):
        _native.require_gfx950(device)
        weight_codes, weight_pitch = _code_rows(weight.codes)
        weight_scales = weight.scales.contiguous()
        added = None if bias is None else bias.contiguous()
        common = (weight_codes.data_ptr(), weight_pitch, weight_scales.data_ptr(), _native.address(added),
                  int(bias is not None and bias.dtype == torch.float32), out.data_ptr())
        stream = _native.retain(device, *tensors)  # (copies of them are this stream's own)
        if quantized:
            codes, pitch = _code_rows(rows)
            scales = x.scales.contiguous()
            status = _native.library().peco_int8_linear(
                codes.data_ptr(), pitch, scales.data_ptr(), *common, count, channels, outputs, _native.dtype_code(dtype),
                stream)
        else:
            source, sizes, strides = outer_axes(x if x.stride(-1) == 1 else x.contiguous())
            codes = _native.dtype_code(x.dtype), _native.dtype_code(dtype)
            size = _workspace_bytes(count, channels, *codes)
            workspace = torch.empty(size, dtype=torch.int8, device=device) if size else None
            status = _native.library().peco_int8_linear_rows(
                source.data_ptr(), _LONG3(*strides), *sizes, codes[0], *common, _native.address(workspace), size, channels,
                outputs, codes[1], stream)
        _native.check(status, "PECO HIP 8-bit projection")
    return out


def _laid_out(codes):
    """A weight's codes [N, K] in rows that the product takes without a copy."""
    if codes.stride(-1) == 1 and codes.stride(0) % 16 == 0 and codes.stride(0) <= 1 << 22 and \
            codes.storage_offset() % 16 == 0:  # (a storage starts on 16 bytes; on the meta device there is no address)
        return codes
    return empty_codes(codes)[0].copy_(codes)


class Int8Linear(torch.nn.Module):
    """A linear layer in 8 bits, for inference: ``int8_linear`` with a weight that is quantized once.

    ``Int8Linear.from_linear(layer)`` takes a ``torch.nn.Linear``'s weight and bias. It takes tensors, or
    QuantizedRows that several layers share; the result has ``dtype``, else autocast's where that is enabled, else the
    tensor's or, for QuantizedRows, the dtype of the layer it was made of.
    """

    def __init__(self, weight: QuantizedRows, bias: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        self.out_features, self.in_features = weight.shape
        self.dtype = dtype
        # (The scales and the bias stay fp32, whatever the module is cast to, and the codes' rows on 16 bytes.)
        self.register_buffer("codes", _laid_out(weight.codes))
        self.register_buffer("scales", weight.scales)
        self.register_buffer("bias", None if bias is None else bias.float())

    @classmethod
    @torch.no_grad()
    def from_linear(cls, layer: torch.nn.Linear) -> "Int8Linear":
        bias = None if layer.bias is None else layer.bias.detach().clone()
        return cls(quantize_rows(layer.weight.detach()), bias, layer.weight.dtype)

    def _apply(self, fn, recurse=True):
        before = self.scales, self.bias
        super()._apply(fn, recurse)
        self.codes = _laid_out(self.codes)  # (a move to another device makes them dense)
        self.scales, self.bias = (now if now is None or now.dtype == torch.float32 else was.to(now.device)
                                  for was, now in zip(before, (self.scales, self.bias)))
        return self

    def result_dtype(self, x) -> torch.dtype:
        """The dtype of ``forward(x)``."""
        if torch.is_autocast_enabled("cuda"):
            return torch.get_autocast_dtype("cuda")
        return self.dtype if isinstance(x, QuantizedRows) else x.dtype

    def forward(self, x, dtype: torch.dtype | None = None):
        return int8_linear(x, QuantizedRows(self.codes, self.scales), self.bias,
                           dtype=self.result_dtype(x) if dtype is None else dtype)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
