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

Arguments are checked and outputs allocated in csrc/binding.cpp.  ``stream``
(a torch.cuda.Stream or a raw handle) is the current stream unless given.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ._launch import native, on_stream

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
    """An empty cache (zeros).  page_size is a power of two up to 4096, dim a
    multiple of 32 up to 1024, heads at most 65536, and num_pages * heads *
    page_size below 2^32."""
    if (num_pages < 0 or not 1 <= heads <= 65536 or not 1 <= page_size <= 4096 or page_size & (page_size - 1)
            or not 32 <= dim <= 1024 or dim % SCALE_BLOCK or num_pages * heads * page_size >= 2 ** 32):
        raise ValueError(f"a cache needs page_size a power of two up to 4096, heads from 1 to 65536, dim a multiple of 32 "
                         f"up to 1024 and num_pages * heads * page_size below 2^32, got num_pages={num_pages}, "
                         f"page_size={page_size}, heads={heads}, dim={dim}")
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    shape = (num_pages, heads, page_size)
    k, v = (torch.zeros((*shape, dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2))
    k_scales, v_scales = (torch.zeros((*shape, dim // SCALE_BLOCK), dtype=torch.uint8, device=device) for _ in range(2))
    return MXFP8Cache(k, v, k_scales, v_scales)


def cache_write(cache: MXFP8Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, stream=None) -> None:
    """Quantize k and v (tokens, heads, dim), bf16 or fp16, into the positions
    ``slots`` (tokens,) int64 of the cache.

    Any token and head strides are read in place (slices of a fused
    projection).  A negative slot skips its token; slots that are written must
    differ from each other.  Every other position keeps its bytes."""
    if stream is None:
        native().cache_write(*cache, k, v, slots)
    else:
        with on_stream(stream, k, v, slots, *cache):
            native().cache_write(*cache, k, v, slots)


def cache_read(cache: MXFP8Cache, page_table: torch.Tensor, starts: torch.Tensor, total: int,
               out_dtype: torch.dtype = torch.bfloat16, out: tuple[torch.Tensor, torch.Tensor] | None = None,
               stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows of a batch, widened and packed: (k, v), each (total, heads, dim).

    ``page_table`` (batch, max_pages) int32, ``starts`` (batch + 1,) int32:
    sequence b has ``starts[b + 1] - starts[b]`` rows, which go to rows
    ``starts[b]`` on; ``total`` is starts[-1], as the host knows it.  Rows
    that no sequence covers are left as they were (uninitialised without a
    given ``out``, a pair of contiguous tensors)."""
    k_out, v_out = (None, None) if out is None else out
    if stream is None:
        return native().cache_read(*cache, page_table, starts, total, out_dtype, k_out, v_out)
    with on_stream(stream, page_table, starts, *cache, k_out, v_out):
        return native().cache_read(*cache, page_table, starts, total, out_dtype, k_out, v_out)


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
    if stream is None:
        out = native().cache_attention(q, *cache, page_table, lengths, scale, return_lse)
    else:
        with on_stream(stream, q, page_table, lengths, *cache):
            out = native().cache_attention(q, *cache, page_table, lengths, scale, return_lse)
    return out if return_lse else out[0]
