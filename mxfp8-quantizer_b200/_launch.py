"""Device, stream and argument handling shared by the 4-bit and cache operators."""

from __future__ import annotations

import contextlib

import torch

from . import _capi

_NOTHING = contextlib.nullcontext()

# Handle of a device's current stream without a Stream object around it: a call
# of these operators costs the host about as much as a small one costs the GPU,
# and torch.cuda.current_stream alone took 2.2 of 16 us.
_current_stream_handle = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)

IN_DTYPES = {torch.bfloat16: _capi.BF16, torch.float16: _capi.FP16}
OUT_DTYPES = {torch.bfloat16: _capi.BF16, torch.float16: _capi.FP16, torch.float32: _capi.F32}


def in_dtype(name: str, dtype: torch.dtype) -> int:
    code = IN_DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"{name} must be torch.bfloat16 or torch.float16, got {dtype}")
    return code


def out_dtype_code(dtype: torch.dtype) -> int:
    code = OUT_DTYPES.get(dtype)
    if code is None:
        raise ValueError("out_dtype must be torch.float32, torch.bfloat16 or torch.float16")
    return code


def on_stream(stream, first: torch.Tensor, *others: torch.Tensor):
    """(context, handle): the context to allocate outputs and launch in, and
    the stream handle.

    All tensors must be on one CUDA device.  ``stream`` None is that device's
    current stream.  Another stream (a torch.cuda.Stream or a raw handle)
    becomes current inside the context, so outputs belong to it, and the
    tensors are recorded on it: their memory is not reused before the launch
    is done, even if the caller drops them.  The caller orders the stream
    after the work that makes the inputs."""
    index = first.get_device()
    if index < 0:
        raise ValueError(f"the operator runs on CUDA tensors, got one on {first.device}")
    for t in others:
        if t.get_device() != index:
            raise ValueError(f"all tensors must be on {first.device}, got one on {t.device}")
    if stream is None:
        context = _NOTHING if torch.cuda.current_device() == index else torch.cuda.device(index)
        return context, _current_stream_handle(index)
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(int(stream), device=first.device)
    if stream.device.index != index:
        raise ValueError(f"the stream is on {stream.device}, the tensors on {first.device}")
    for t in (first, *others):
        t.record_stream(stream)
    return torch.cuda.stream(stream), stream.cuda_stream
