"""4-bit microscaling beside the MXFP8 quantizer: quantize, dequantize and the
product of two MXFP4 matrices (C ABI in include/mxfp4.h).

An MXFP4 matrix is a pair ``(q, s)``: ``q`` (rows, cols / 2) uint8 holds two
E2M1 codes a byte (the even column in the low four bits), ``s`` one UE8M0 byte
per 1x32 block along the columns, in the chunk layout of
``packed_scale_storage_bytes(rows, cols)`` that ``quantize`` writes too.  The
reference quantizes to E4M3 only, so nothing here has a counterpart there.

Arguments are checked and outputs allocated in csrc/binding.cpp.  ``stream``
(a torch.cuda.Stream or a raw handle) is the current stream unless given.
"""

from __future__ import annotations

import torch

from ._launch import native, on_stream

FP4_E2M1_MAX = 6.0


def quantize_mxfp4(x: torch.Tensor, q: torch.Tensor | None = None, s: torch.Tensor | None = None, stream=None):
    """Quantize a CUDA (m, k) bf16/fp16 tensor to MXFP4; returns (q, s).

    The scale of a block is the smallest power of two that keeps its largest
    magnitude within 6, the codes are rounded to nearest (ties to even); a
    block that holds an inf or a NaN decodes to NaN.  Columns are padded with
    zeros to a multiple of 32.  ``x`` may have any row stride and offset; one
    whose last dimension is not contiguous is copied first.  Preallocated
    ``q`` (m, ceil(k/32)*16) and ``s`` are written in place."""
    if stream is None:
        return native().quantize_mxfp4(x, q, s)
    with on_stream(stream, x, q, s):
        return native().quantize_mxfp4(x, q, s)


def dequantize_mxfp4(q: torch.Tensor, s: torch.Tensor, out_dtype: torch.dtype = torch.float32, stream=None):
    """MXFP4 payload + packed UE8M0 scales -> out_dtype (bf16, fp16 or fp32)."""
    if stream is None:
        return native().dequantize_mxfp4(q, s, out_dtype)
    with on_stream(stream, q, s):
        return native().dequantize_mxfp4(q, s, out_dtype)


def mxfp4_gemm(a_q: torch.Tensor, b_q: torch.Tensor, a_s: torch.Tensor, b_s: torch.Tensor,
               out_dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """C (m, n) = A B^T of two MXFP4 matrices A (m, k) and B (n, k), summed in
    fp32 and rounded once to out_dtype (fp32, bf16 or fp16): the 4-bit form of
    ``blockscaled_gemm``, on this library's own kernel.

    ``a_q``/``a_s`` and ``b_q``/``b_s`` are what ``quantize_mxfp4`` returns
    (scale bytes of the padding must not be 255; it writes 0).  A given
    ``out`` (m, n), row-major with any row stride, is written in place and
    sets the output type; it must not overlap the operands."""
    if stream is None:
        return native().mxfp4_gemm(a_q, b_q, a_s, b_s, out_dtype, out)
    with on_stream(stream, a_q, b_q, a_s, b_s, out):
        return native().mxfp4_gemm(a_q, b_q, a_s, b_s, out_dtype, out)
