"""Attention with a sliding window and sinks on gfx950 MFMA: forward and backward.

For clips that are generated or fine-tuned piece by piece: a token sees the tokens of a window around it (causal
or to both sides) and the first tokens of its sequence (the prompt's, say), which stay visible to every later one.
``paged.paged_attention`` is the same attention over a cache.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _native


def rows16(t):
    """t with adjacent channels and every row on 16 bytes (a copy when it is laid out otherwise)."""
    *outer, inner = t.stride()
    if inner == 1 and t.data_ptr() % 16 == 0:
        low = 0
        for s in outer:
            low |= s
        if low % 8 == 0:
            return t
    return t.clone(memory_format=torch.contiguous_format)


def strides_of(*tensors):
    """The strides of all but the last axis of the tensors, as the C-ABI's host array."""
    values = []
    for t in tensors:
        values += t.stride()[:-1]
    return _long_array(len(values))(*values)


@functools.lru_cache(maxsize=None)
def _long_array(n):
    return ctypes.c_int64 * n


@functools.lru_cache(maxsize=1024)
def workspace_floats(entry, device_index, *sizes):
    """A workspace size query's answer; it depends on the sizes and on the device's compute units alone."""
    return getattr(_native.library(), entry)(*sizes)


def raise_error(error, what):
    if error:
        message = _native.library().peco_attention_error_string(error).decode("utf-8", errors="replace")
        raise RuntimeError(f"PECO HIP {what} launch failed: {message} ({error})")


def check_mask(window, sinks, scale, dim):
    """(left, right, sinks, scale) as the kernels take them: limits in [-1, 2^30], a positive scale."""
    if not isinstance(window, (tuple, list)) or len(window) != 2 or \
            any(isinstance(n, bool) or not isinstance(n, int) or n < -1 for n in window):
        raise ValueError("window must be (left, right), nonnegative integers or -1 for no limit")
    if isinstance(sinks, bool) or not isinstance(sinks, int) or sinks < 0:
        raise ValueError("sinks must be a nonnegative integer")
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:
        raise ValueError("scale must be a positive finite number")
    most = 1 << 30
    return min(window[0], most), min(window[1], most), min(sinks, most), scale


def _check(q, k, v, lengths):
    tensors = (q, k, v) if lengths is None else (q, k, v, lengths)
    if not all(isinstance(t, torch.Tensor) for t in tensors):
        raise TypeError("All window attention inputs must be torch tensors")
    if q.ndim != 4 or k.ndim != 4 or v.shape != k.shape:
        raise ValueError("Expected Q [B,HQ,SQ,D] and equal-shaped K/V [B,HK,SK,D]")
    batch, heads, sq, dim = q.shape
    if k.shape[0] != batch or k.shape[3] != dim:
        raise ValueError("Q and K/V batch and feature dimensions must match")
    if k.shape[1] < 1 or heads < 1 or heads % k.shape[1]:
        raise ValueError("the query heads must be a multiple of the key heads")
    if dim not in (64, 128):
        raise ValueError("HIP attention supports head dimensions 64 and 128")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("Q/K/V must share dtype torch.float16 or torch.bfloat16")
    if lengths is not None:
        if sq != k.shape[2]:
            raise ValueError("lengths needs as many queries as keys")
        if lengths.dtype != torch.int32 or lengths.shape != (batch,):
            raise TypeError("lengths must be int32 [B]")
    device = q.device
    if not q.is_cuda or k.device != device or v.device != device or (lengths is not None and lengths.device != device):
        raise ValueError("All window attention inputs must reside on the same GPU device")
    if not _native.plain_tensors(*tensors):
        raise RuntimeError("window_attention takes ordinary tensors (no tracing, transforms or tangents)")
    if max(sq, k.shape[2]) >= 1 << 30:
        raise ValueError("sequences must be shorter than 2^30")


def _forward(q, k, v, lengths, left, right, sinks, scale, stats):
    """(output, row references, log2 of the row sums, rest of the output); the last three None without ``stats``."""
    batch, heads, sq, dim = q.shape
    kv_heads, sk = k.shape[1:3]
    out = torch.empty_like(q)
    row_max = row_log = rest = workspace = None
    if q.numel() == 0:
        return out, row_max, row_log, rest
    if sk == 0:
        return out.zero_(), row_max, row_log, rest
    device, address = q.device, _native.address
    with _native.on_device(device):
        _native.require_gfx950(device)
        q, k, v = rows16(q), rows16(k), rows16(v)
        target = out if rows16(out) is out else torch.empty(out.shape, dtype=out.dtype, device=device)
        if stats:
            row_max, row_log = torch.empty((2, batch, heads, sq), dtype=torch.float32, device=device).unbind()
            rest = torch.empty((batch, heads, sq, dim), dtype=q.dtype, device=device)
        shape = (batch, heads, kv_heads, sq, sk, left, right, sinks)
        floats = workspace_floats("peco_window_attention_workspace_size", device.index, *shape, dim)
        if floats:
            workspace = torch.empty(floats, dtype=torch.float32, device=device)
        raise_error(_native.library().peco_window_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), target.data_ptr(), strides_of(q, k, v, target),
            address(lengths), address(row_max), address(row_log), address(rest), address(workspace), floats, *shape, scale,
            dim, _native.dtype_code(q.dtype), _native.retain(device, q, k, v, lengths)), "window attention")
        return (out if target is out else out.copy_(target)), row_max, row_log, rest


def _backward(q, k, v, out, row_max, row_log, rest, lengths, grad, left, right, sinks, scale):
    if not _native.plain_gradient(grad):
        raise RuntimeError("the gradient of window_attention's output must be an ordinary tensor (no tracing, transforms, "
                           "batches or tangents)")
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    if row_max is None:  # no query or no key: nothing is seen
        return dq.zero_(), dk.zero_(), dv.zero_()
    batch, heads, sq, dim = q.shape
    device, address = q.device, _native.address
    with _native.on_device(device):
        given = [rows16(t) for t in (q, k, v, out, grad)]
        shape = (batch, heads, k.shape[1], sq, k.shape[2], left, right, sinks)
        code = _native.dtype_code(q.dtype)
        floats = workspace_floats("peco_window_attention_grad_workspace_size", device.index, *shape, dim, code)
        workspace = torch.empty(floats, dtype=torch.float32, device=device)
        raise_error(_native.library().peco_window_attention_grad(
            *[t.data_ptr() for t in given], dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
            strides_of(*given, dq, dk, dv), address(lengths), row_max.data_ptr(), row_log.data_ptr(), rest.data_ptr(),
            workspace.data_ptr(), floats, *shape, scale, dim, code,
            _native.retain(device, *given, lengths, row_max, row_log, rest)), "window attention gradient")
    return dq, dk, dv


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, mask):
        out, row_max, row_log, rest = _forward(q, k, v, lengths, *mask, True)
        ctx.save_for_backward(q, k, v, lengths, out, row_max, row_log, rest)
        ctx.mask = mask
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        q, k, v, lengths, out, row_max, row_log, rest = ctx.saved_tensors
        return (*_backward(q, k, v, out, row_max, row_log, rest, lengths, grad, *ctx.mask), None, None)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window, sinks: int = 0, *,
                     lengths: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """softmax(scale Q K^T) V over the keys that each query sees.

    Q [B,HQ,SQ,D] and K/V [B,HK,SK,D], fp16 or bf16, D 64 or 128, any strides (tensors whose rows do not lie on
    16 bytes with adjacent channels are copied first); HQ a multiple of HK, query head h reads key head
    h // (HQ / HK). Queries and keys end together: query i stands at position p = i + SK - SQ and sees key j when
    j <= p + right and (j >= p - left or j < sinks), with ``window = (left, right)``, -1 for no limit: (-1, 0) is
    causal, (n - 1, 0) a causal window of n tokens, (n, n) one to both sides. A query that sees no key gives 0.
    ``lengths`` (int32 [B], needs SQ == SK): valid tokens of each sequence of a right-padded batch; later keys are
    not seen, later rows give 0 and take no gradient, whatever they hold. ``scale`` defaults to 1 / sqrt(D).
    The result has the strides of ``empty_like(q)``. Scores, softmax statistics and all sums are fp32; the weights
    are rounded to the dtype for their product with V (fp16: those below 2^-25 of a row's largest add nothing) and the
    result once. A query whose scores are all -inf gives 0, as one that sees no key.

    Differentiable once in Q, K and V. Weights and dS are rounded to the dtype for their products, which leaves the
    gradients 1.4 to 1.5 times as far off as their own rounding does; calls whose queries see at most 8 keys, or of at
    most 2^20 pairs of a query and a key that it may see, keep them at full precision. The gradient of the result must be
    an ordinary tensor (no batch of gradients, no tangent). A backward pass may be
    captured into a HIP graph while no eager graph of the same leaves is alive (torch's engine would accumulate
    their gradients on that graph's stream and end the process).
    """
    _check(q, k, v, lengths)
    mask = check_mask(window, sinks, scale, q.shape[3])
    lengths = None if lengths is None else lengths.contiguous()
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v)):
        return _WindowAttention.apply(q, k, v, lengths, mask)
    return _forward(q, k, v, lengths, *mask, False)[0]
