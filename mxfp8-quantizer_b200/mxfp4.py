"""4-bit microscaling beside the MXFP8 quantizer: quantize, dequantize and the
product of two MXFP4 matrices (C ABI in include/mxfp4.h).

An MXFP4 matrix is a pair ``(q, s)``: ``q`` (rows, cols / 2) uint8 holds two
E2M1 codes a byte (the even column in the low four bits), ``s`` one UE8M0 byte
per 1x32 block along the columns, in the chunk layout of
``packed_scale_storage_bytes(rows, cols)`` that ``quantize`` writes too.  The
reference quantizes to E4M3 only, so nothing here has a counterpart there.
"""

from __future__ import annotations

import torch

from . import _capi
from ._launch import in_dtype, on_stream, out_dtype_code

FP4_E2M1_MAX = 6.0
_PAYLOAD_DTYPES = (torch.uint8, torch.int8, torch.float4_e2m1fn_x2)


def _check_payload(name: str, q: torch.Tensor) -> tuple[int, int]:
    """(rows, cols) of an MXFP4 payload."""
    if q.dim() != 2 or q.dtype not in _PAYLOAD_DTYPES or (q.stride()[1] != 1 and q.shape[1] > 1):
        raise ValueError(f"{name} must be a row-major matrix of bytes, got {tuple(q.shape)} {q.dtype}")
    rows, row_bytes = q.shape
    if row_bytes % 16:
        raise ValueError(f"{name} must have a multiple of 32 columns (16 bytes), got {2 * row_bytes}")
    return rows, 2 * row_bytes


def _check_scales(name: str, s: torch.Tensor) -> None:
    """The library checks the size."""
    if s.element_size() != 1 or not s.is_contiguous():
        raise ValueError(f"{name} must be a contiguous buffer of bytes")


def _row_stride(t: torch.Tensor) -> int:
    """Row stride, also of a matrix whose single row carries none."""
    rows, cols = t.shape
    row = t.stride()[0]
    return row if rows > 1 else max(row, cols)


def quantize_mxfp4(x: torch.Tensor, q: torch.Tensor | None = None, s: torch.Tensor | None = None, stream=None):
    """Quantize a CUDA (m, k) bf16/fp16 tensor to MXFP4; returns (q, s).

    The scale of a block is the smallest power of two that keeps its largest
    magnitude within 6, the codes are rounded to nearest (ties to even); a
    block that holds an inf or a NaN decodes to NaN.  Columns are padded with
    zeros to a multiple of 32.  ``x`` may have any row stride and offset; one
    whose last dimension is not contiguous is copied first.  Preallocated
    ``q`` (m, ceil(k/32)*16) and ``s`` are written in place."""
    if x.dim() != 2:
        raise ValueError(f"X must be 2-D, got shape {tuple(x.shape)}")
    code = in_dtype("X", x.dtype)
    m, k = x.shape
    q_cols = -(-k // 32) * 32
    context, handle = on_stream(stream, x, *(t for t in (q, s) if t is not None))
    with context:
        row, col = x.stride()
        if (col != 1 and k > 1) or (m > 1 and row < k):
            x = x.contiguous()
        if q is None:
            q = torch.empty(m, q_cols // 2, dtype=torch.uint8, device=x.device)
        elif _check_payload("q", q) != (m, q_cols):
            raise ValueError(f"q must be ({m}, {q_cols // 2}) bytes, got {tuple(q.shape)}")
        need = -(-m // 128) * 128 * (-(-q_cols // 128) * 4)
        if s is None:
            s = torch.empty(need, dtype=torch.uint8, device=x.device)
        else:
            _check_scales("s", s)
        _capi.fp4_quantize(x.data_ptr(), code, m, k, _row_stride(x), q.data_ptr(), _row_stride(q), s.data_ptr(),
                           s.numel(), handle)
    return q, s


def dequantize_mxfp4(q: torch.Tensor, s: torch.Tensor, out_dtype: torch.dtype = torch.float32, stream=None):
    """MXFP4 payload + packed UE8M0 scales -> out_dtype (bf16, fp16 or fp32)."""
    rows, cols = _check_payload("q", q)
    _check_scales("s", s)
    code = out_dtype_code(out_dtype)
    context, handle = on_stream(stream, q, s)
    with context:
        out = torch.empty(rows, cols, dtype=out_dtype, device=q.device)
        _capi.fp4_dequantize(q.data_ptr(), rows, cols, _row_stride(q), s.data_ptr(), s.numel(), out.data_ptr(), code,
                             cols, handle)
    return out


def mxfp4_gemm(a_q: torch.Tensor, b_q: torch.Tensor, a_s: torch.Tensor, b_s: torch.Tensor,
               out_dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """C (m, n) = A B^T of two MXFP4 matrices A (m, k) and B (n, k), summed in
    fp32 and rounded once to out_dtype (fp32, bf16 or fp16): the 4-bit form of
    ``blockscaled_gemm``, on this library's own kernel.

    ``a_q``/``a_s`` and ``b_q``/``b_s`` are what ``quantize_mxfp4`` returns
    (scale bytes of the padding must not be 255; it writes 0).  A given
    ``out`` (m, n), row-major with any row stride, is written in place and
    sets the output type; it must not overlap the operands."""
    m, k = _check_payload("a_q", a_q)
    n, k_b = _check_payload("b_q", b_q)
    if k != k_b:
        raise ValueError(f"a_q and b_q must have the same number of columns, got {k} and {k_b}")
    _check_scales("a_s", a_s)
    _check_scales("b_s", b_s)
    if out is not None:
        if out.dim() != 2 or tuple(out.shape) != (m, n) or (out.stride(1) != 1 and n > 1):
            raise ValueError(f"out must be a row-major ({m}, {n}) matrix, got {tuple(out.shape)}")
        out_dtype = out.dtype
    code = out_dtype_code(out_dtype)
    context, handle = on_stream(stream, a_q, b_q, a_s, b_s, *(() if out is None else (out,)))
    with context:
        if out is None:
            out = torch.empty(m, n, dtype=out_dtype, device=a_q.device)
        _capi.fp4_gemm(a_q.data_ptr(), m, _row_stride(a_q), a_s.data_ptr(), a_s.numel(), b_q.data_ptr(), n,
                       _row_stride(b_q), b_s.data_ptr(), b_s.numel(), k, out.data_ptr(), code, _row_stride(out), handle)
    return out
