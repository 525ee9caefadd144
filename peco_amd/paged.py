"""A paged key/value cache on gfx950: new tokens' keys and values appended, new queries' attention over it.

A cache is two tensors of pages, K and V [pages, heads, page, D] (any strides with adjacent channels), and per
sequence a row of page numbers: token t of sequence b is slot t % page of page ``page_table[b, t // page]``. A call
takes the new tokens of a batch of sequences in a row, sequence b's at ``offsets[b]`` to ``offsets[b + 1]``, and
every sequence's number of tokens with the new ones, ``lengths``. All of these are on the GPU and are not read by
the host, so a captured graph serves any batch that fits its sizes.
"""
from __future__ import annotations

import torch

from . import _native, rotary as rotary_module
from .window import check_mask, raise_error, rows16, strides_of, workspace_floats


def _check_cache(k_pages, v_pages, page_table, offsets, lengths, rows, name):
    tensors = (rows, k_pages, v_pages, page_table, offsets, lengths)
    if not all(isinstance(t, torch.Tensor) for t in tensors):
        raise TypeError("All paged cache inputs must be torch tensors")
    if k_pages.ndim != 4 or v_pages.shape != k_pages.shape or min(k_pages.shape[:3]) < 1:
        raise ValueError("Expected equal-shaped K/V pages [pages,HK,page,D] that are not empty")
    if rows.ndim != 3 or rows.shape[2] != k_pages.shape[3]:
        raise ValueError(f"Expected {name} [tokens,heads,D] with the pages' feature dimension")
    if k_pages.shape[3] not in (64, 128):
        raise ValueError("HIP attention supports head dimensions 64 and 128")
    if rows.dtype not in (torch.float16, torch.bfloat16) or k_pages.dtype != rows.dtype or v_pages.dtype != rows.dtype:
        raise TypeError(f"{name} and the pages must share dtype torch.float16 or torch.bfloat16")
    if page_table.ndim != 2 or min(page_table.shape) < 1:
        raise ValueError("page_table must have shape [sequences,entries] and not be empty")
    if offsets.shape != (page_table.shape[0] + 1,) or lengths.shape != (page_table.shape[0],):
        raise ValueError("offsets and lengths must have shapes [sequences + 1] and [sequences]")
    if page_table.dtype != torch.int32 or offsets.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise TypeError("page_table, offsets and lengths must be int32")
    device = rows.device
    if not rows.is_cuda or k_pages.device != device or v_pages.device != device or page_table.device != device or \
            offsets.device != device or lengths.device != device:
        raise ValueError("All paged cache inputs must reside on the same GPU device")
    if not _native.plain_tensors(*tensors):
        raise RuntimeError("a paged cache takes ordinary tensors (no tracing, transforms or tangents)")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (rows, k_pages, v_pages)):
        raise RuntimeError("a paged cache supports inference only; use torch.no_grad()")
    for t in (k_pages, v_pages):
        a, b, c, inner = t.stride()
        if inner != 1 or (a | b | c) % 8 or t.data_ptr() % 16:
            raise ValueError("pages must have adjacent channels and rows on 16 bytes")
    if page_table.shape[1] * k_pages.shape[2] >= 1 << 30 or rows.shape[0] >= 1 << 30:
        raise ValueError("sequences must be shorter than 2^30")


_NO_PLAN = (None, 0, 0, 0, None, None, 0, 0, 0)


def _repeats_rows(t):
    return any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape))


def append_pages(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 page_table: torch.Tensor, offsets: torch.Tensor, lengths: torch.Tensor, *,
                 rotary: rotary_module.RotaryPositions | None = None) -> None:
    """Write new tokens' keys and values k, v [tokens,HK,D] to their places in the cache.

    Token i of n new ones of sequence b goes to place lengths[b] - n + i (``lengths`` count the new tokens).
    With ``rotary`` (positions [axes,tokens]) the keys are turned first, as ``rotary.rotary_axes`` turns them.
    Tokens of no sequence, places outside the table and pages outside [0, pages) are passed over; two places that
    share a page's row (a page given twice) are written in no order.
    """
    _check_cache(k_pages, v_pages, page_table, offsets, lengths, k, "k and v")
    if not isinstance(v, torch.Tensor) or v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
        raise ValueError("k and v must be tensors of one shape, dtype and device")
    if not _native.plain_tensors(v) or (torch.is_grad_enabled() and v.requires_grad):
        raise RuntimeError("a paged cache supports inference only; use torch.no_grad()")
    tokens, heads, dim = k.shape
    pages, kv_heads, page, _ = k_pages.shape
    if heads != kv_heads:
        raise ValueError("k and v must have the pages' heads")
    if _repeats_rows(k_pages) or _repeats_rows(v_pages):
        raise ValueError("pages that are written must not be expanded")
    positions, plan = None, _NO_PLAN
    if rotary is not None:
        if not isinstance(rotary, rotary_module.RotaryPositions):
            raise TypeError("rotary must be a RotaryPositions")
        positions = rotary_module.check_positions(rotary.axes, rotary.positions, 1, tokens, dim, k.device)
        plan = rotary_module.plan_arguments(rotary.axes, positions)
    if tokens == 0:
        return
    device = k.device
    with _native.on_device(device):
        _native.require_gfx950(device)
        k, v, table = rows16(k), rows16(v), page_table if page_table.stride(1) == 1 else page_table.contiguous()
        offsets, lengths = offsets.contiguous(), lengths.contiguous()
        _native.check(_native.library().peco_append_pages(
            k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), strides_of(k, v, k_pages, v_pages),
            table.data_ptr(), table.stride(0), offsets.data_ptr(), lengths.data_ptr(), *plan, table.shape[0], heads,
            tokens, pages, page, table.shape[1], dim, _native.dtype_code(k.dtype),
            _native.retain(device, k, v, k_pages, v_pages, table, offsets, lengths, positions)), "PECO HIP append to pages")


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    offsets: torch.Tensor, lengths: torch.Tensor, *, window: int = -1, sinks: int = 0,
                    scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of new tokens q [tokens,HQ,D] over the cache, causal, with ``window.window_attention``'s mask.

    The new tokens are the last ones of their sequences and are in the cache already (``append_pages``): new token
    i of n of a sequence of ``lengths[b]`` tokens stands at p = lengths[b] - n + i and sees token j when j <= p and
    (j >= p - window or j < sinks); ``window`` -1 is without limit. HQ is a multiple of the pages' heads HK, query
    head h reads key head h // (HQ / HK). Keys on a page whose number in ``page_table`` is outside [0, pages) (one
    that left the window and was given back, say) are not seen. A query that sees no key gives 0. ``offsets``
    ascend; ``lengths`` are taken within [0, table's tokens]. Rows of q of no sequence, those behind
    ``offsets[-1]`` of a padded batch, give 0, or with ``out`` (a tensor like q) are left there as they were. Roundings
    are ``window.window_attention``'s: fp32 but for the weights in their product with V and the result.
    """
    _check_cache(k_pages, v_pages, page_table, offsets, lengths, q, "q")
    tokens, heads, dim = q.shape
    pages, kv_heads, page, _ = k_pages.shape
    if heads < 1 or heads % kv_heads:
        raise ValueError("the query heads must be a multiple of the pages' heads")
    left, _, sinks, scale = check_mask((window, 0), sinks, scale, dim)
    if out is not None:
        if not isinstance(out, torch.Tensor) or out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
            raise ValueError("out must be a tensor like q")
        if not _native.plain_tensors(out) or (torch.is_grad_enabled() and out.requires_grad):
            raise RuntimeError("out must be an ordinary tensor without gradient")
        if rows16(out) is not out or _repeats_rows(out):
            raise ValueError("out must have adjacent channels and rows on 16 bytes and not be expanded")
    result = torch.empty((tokens, heads, dim), dtype=q.dtype, device=q.device) if out is None else out
    if tokens == 0:
        return result
    device = q.device
    with _native.on_device(device):
        _native.require_gfx950(device)
        q, table = rows16(q), page_table if page_table.stride(1) == 1 else page_table.contiguous()
        offsets, lengths = offsets.contiguous(), lengths.contiguous()
        batch, width = table.shape
        floats = workspace_floats("peco_paged_attention_workspace_size", device.index, batch, heads, kv_heads, tokens, width,
                                  page, left, sinks, dim)
        workspace = torch.empty(floats, dtype=torch.float32, device=device) if floats else None
        # (q and the output count head before token.)
        strides = strides_of(q.transpose(0, 1), k_pages, v_pages, result.transpose(0, 1))
        raise_error(_native.library().peco_paged_attention(
            q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), result.data_ptr(), strides, table.data_ptr(),
            table.stride(0), offsets.data_ptr(), lengths.data_ptr(), int(out is None), _native.address(workspace), floats,
            batch, heads, kv_heads, tokens, pages, page, width, left, sinks, scale, dim, _native.dtype_code(q.dtype),
            _native.retain(device, q, k_pages, v_pages, out, table, offsets, lengths)), "paged attention")
    return result
