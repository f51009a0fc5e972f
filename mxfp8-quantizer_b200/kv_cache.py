"""Key/value cache in MXFP8: rows quantized into pages as they are written,
read back widened, and attended to by single query tokens (C ABI in
include/mxfp8_cache.h).

A cache holds a position's K and V row of every KV head as E4M3 bytes with one
UE8M0 scale per 32 elements, by the recipe of ``quantize``: 1 + 1/32 bytes an
element instead of 2.  Positions are numbered ``page * page_size + offset``;
a sequence is a row of a page table.  The reference has no cache, so nothing
here has a counterpart there.

Pages, slots and lengths stay on the device and are checked there: an index
outside the cache is never followed, and shows up as bit 64 of
``check_cuda_launch_errors`` / ``_capi.device_status``.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _capi
from ._launch import in_dtype, on_stream, out_dtype_code

SCALE_BLOCK = 32


class MXFP8Cache(NamedTuple):
    """The four buffers of a cache, contiguous and on one device:
    ``k``, ``v`` (num_pages, heads, page_size, dim) float8_e4m3fn and
    ``k_scales``, ``v_scales`` (num_pages, heads, page_size, dim / 32) uint8."""

    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor


def allocate_cache(num_pages: int, page_size: int, heads: int, dim: int, device=None) -> MXFP8Cache:
    """An empty cache (zeros).  page_size is a power of two, dim a multiple of 32."""
    if num_pages < 0 or heads < 1 or page_size < 1 or page_size & (page_size - 1) or dim < 32 or dim % SCALE_BLOCK:
        raise ValueError(f"a cache needs page_size a power of two, heads >= 1 and dim a multiple of 32, got "
                         f"num_pages={num_pages}, page_size={page_size}, heads={heads}, dim={dim}")
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    shape = (num_pages, heads, page_size)
    k, v = (torch.zeros((*shape, dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2))
    k_scales, v_scales = (torch.zeros((*shape, dim // SCALE_BLOCK), dtype=torch.uint8, device=device) for _ in range(2))
    return MXFP8Cache(k, v, k_scales, v_scales)


def _describe(cache: MXFP8Cache) -> _capi.Cache:
    k, v, k_scales, v_scales = cache
    shape = k.shape
    if len(shape) != 4 or k.element_size() != 1 or v.element_size() != 1 or v.shape != shape:
        raise ValueError(f"k and v must be (num_pages, heads, page_size, dim) bytes, got {tuple(shape)} {k.dtype} and "
                         f"{tuple(v.shape)} {v.dtype}")
    pages, heads, page_size, dim = shape
    scale_shape = (pages, heads, page_size, dim // SCALE_BLOCK)
    if dim % SCALE_BLOCK or k_scales.shape != scale_shape or v_scales.shape != scale_shape:
        raise ValueError(f"the scales must be {scale_shape} for dim a multiple of 32, got {tuple(k_scales.shape)} and "
                         f"{tuple(v_scales.shape)}")
    if k_scales.element_size() != 1 or v_scales.element_size() != 1:
        raise ValueError("the scales must be bytes")
    if not (k.is_contiguous() and v.is_contiguous() and k_scales.is_contiguous() and v_scales.is_contiguous()):
        raise ValueError("the cache's buffers must be contiguous")
    return _capi.Cache(k.data_ptr(), v.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), pages, heads, page_size,
                       dim)


def _check_index(name: str, t: torch.Tensor, dtype: torch.dtype, dims: int) -> None:
    if t.dtype != dtype or t.dim() != dims or (t.stride()[-1] != 1 and t.shape[-1] > 1):
        raise ValueError(f"{name} must be a {dims}-D {dtype} tensor with a contiguous last dimension, got "
                         f"{tuple(t.shape)} {t.dtype}")


def _check_rows(name: str, t: torch.Tensor, heads: int | None, dim: int) -> None:
    shape = t.shape
    if len(shape) != 3 or shape[2] != dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name} must be (rows, {'heads' if heads is None else heads}, {dim}), got {tuple(shape)}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with a contiguous last dimension."""
    return t if t.stride()[2] == 1 else t.contiguous()


def _table_stride(table: torch.Tensor) -> int:
    batch, width = table.shape
    return table.stride()[0] if batch > 1 else width


def cache_write(cache: MXFP8Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, stream=None) -> None:
    """Quantize k and v (tokens, heads, dim), bf16 or fp16, into the positions
    ``slots`` (tokens,) int64 of the cache.

    Any token and head strides are read in place (slices of a fused
    projection).  A negative slot skips its token; slots that are written must
    differ from each other.  Every other position keeps its bytes."""
    shape = _describe(cache)
    _check_rows("k", k, shape.heads, shape.dim)
    _check_rows("v", v, shape.heads, shape.dim)
    _check_index("slots", slots, torch.int64, 1)
    tokens = k.shape[0]
    if v.shape[0] != tokens or slots.shape[0] != tokens or v.dtype != k.dtype:
        raise ValueError(f"k, v and slots must have the same number of tokens and k and v one type, got "
                         f"{tuple(k.shape)} {k.dtype}, {tuple(v.shape)} {v.dtype}, {tuple(slots.shape)}")
    code = in_dtype("k", k.dtype)
    context, handle = on_stream(stream, k, v, slots, *cache)
    with context:
        k, v = _rows(k), _rows(v)
        k_token, k_head, _ = k.stride()
        v_token, v_head, _ = v.stride()
        _capi.cache_write(shape, k.data_ptr(), k_token, k_head, v.data_ptr(), v_token, v_head, code, tokens,
                          slots.data_ptr(), handle)


def cache_read(cache: MXFP8Cache, page_table: torch.Tensor, starts: torch.Tensor, total: int,
               out_dtype: torch.dtype = torch.bfloat16, out: tuple[torch.Tensor, torch.Tensor] | None = None,
               stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows of a batch, widened and packed: (k, v), each (total, heads, dim).

    ``page_table`` (batch, max_pages) int32, ``starts`` (batch + 1,) int32:
    sequence b has ``starts[b + 1] - starts[b]`` rows, which go to rows
    ``starts[b]`` on; ``total`` is starts[-1], as the host knows it.  Rows
    that no sequence covers are left as they were (uninitialised without a
    given ``out``, a pair of contiguous tensors)."""
    shape = _describe(cache)
    _check_index("page_table", page_table, torch.int32, 2)
    _check_index("starts", starts, torch.int32, 1)
    batch, max_pages = page_table.shape
    if starts.shape[0] != batch + 1:
        raise ValueError(f"starts must have batch + 1 = {batch + 1} values, got {starts.shape[0]}")
    if total < 0:
        raise ValueError(f"total must be >= 0, got {total}")
    want = (total, shape.heads, shape.dim)
    if out is not None:
        for t in out:
            if tuple(t.shape) != want or not t.is_contiguous() or t.dtype != out[0].dtype:
                raise ValueError(f"out must be a pair of contiguous {want} tensors of one type")
        out_dtype = out[0].dtype
    code = out_dtype_code(out_dtype)
    context, handle = on_stream(stream, page_table, starts, *cache, *(out or ()))
    with context:
        if out is None:
            k_out = torch.empty(*want, dtype=out_dtype, device=page_table.device)
            out = k_out, torch.empty_like(k_out)
        _capi.cache_read(shape, page_table.data_ptr(), _table_stride(page_table), max_pages, batch, starts.data_ptr(),
                         total, out[0].data_ptr(), out[1].data_ptr(), code, handle)
    return out[0], out[1]


def cache_attention(q: torch.Tensor, cache: MXFP8Cache, page_table: torch.Tensor, lengths: torch.Tensor,
                    scale: float | None = None, return_lse: bool = False, stream=None):
    """Attention of one query token per sequence over its cached positions.

    ``q`` (batch, q_heads, dim) bf16 or fp16, q_heads a multiple of the
    cache's heads (query heads h * group .. share KV head h); ``page_table``
    (batch, max_pages) int32; ``lengths`` (batch,) int32.  Returns out
    (batch, q_heads, dim) of q's type, and with ``return_lse`` also the
    fp32 (batch, q_heads) log of the softmax's sum, for joining with other
    parts of a context.  A length of 0 gives zeros and -inf.  ``scale`` is
    1/sqrt(dim) unless given.  dim is 64, 128, 192 or 256 and page_size at least 2."""
    shape = _describe(cache)
    _check_rows("q", q, None, shape.dim)
    _check_index("page_table", page_table, torch.int32, 2)
    _check_index("lengths", lengths, torch.int32, 1)
    batch, q_heads = q.shape[0], q.shape[1]
    if page_table.shape[0] != batch or lengths.shape[0] != batch:
        raise ValueError(f"page_table and lengths must have q's batch of {batch}, got {tuple(page_table.shape)} and "
                         f"{tuple(lengths.shape)}")
    if q_heads < 1 or q_heads % shape.heads:
        raise ValueError(f"q must have a multiple of the cache's {shape.heads} heads, got {q_heads}")
    if shape.dim not in (64, 128, 192, 256) or shape.page_size < 2:
        raise ValueError(f"attention needs dim 64, 128, 192 or 256 and page_size >= 2, got {shape.dim} and "
                         f"{shape.page_size}")
    code = in_dtype("q", q.dtype)
    context, handle = on_stream(stream, q, page_table, lengths, *cache)
    with context:
        q = _rows(q)
        q_batch, q_head, _ = q.stride()
        device = q.device
        out = torch.empty(batch, q_heads, shape.dim, dtype=q.dtype, device=device)
        lse = torch.empty(batch, q_heads, dtype=torch.float32, device=device) if return_lse else None
        size = _capi.cache_attention_workspace(shape, batch, q_heads)
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        _capi.cache_attention(shape, q.data_ptr(), q_batch, q_head, code, batch, q_heads, page_table.data_ptr(),
                              _table_stride(page_table), page_table.shape[1], lengths.data_ptr(),
                              1.0 / math.sqrt(shape.dim) if scale is None else scale, out.data_ptr(),
                              0 if lse is None else lse.data_ptr(), workspace.data_ptr(), size, handle)
    return (out, lse) if return_lse else out
