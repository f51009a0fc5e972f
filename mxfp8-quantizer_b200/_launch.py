"""The compiled binding of the 4-bit and cache operators (csrc/binding.cpp), and
the streams that they are given."""

from __future__ import annotations

import contextlib
import ctypes
import importlib.util
import threading

import torch

from . import _capi

NATIVE_PATH = _capi.PKG_DIR / "_native.so"

_lock = threading.Lock()
_native = None


def native():
    """The binding, loaded once and given the library's entries; there is no fallback."""
    global _native
    if _native is not None:
        return _native
    with _lock:
        if _native is not None:
            return _native
        if not NATIVE_PATH.exists():
            raise _capi.ExtensionMissing(
                f"{NATIVE_PATH} is not built; run `python {_capi.PKG_DIR.name}/build.py` (or __graft_entry__.build())")
        lib = _capi.lib()
        spec = importlib.util.spec_from_file_location("_native", NATIVE_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        entries = {name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value
                   for name in _capi.FP4_EXPORTS + _capi.CACHE_EXPORTS}
        module.bind(entries, _capi.check)
        _native = module
        return module


@contextlib.contextmanager
def on_stream(stream, *tensors):
    """Make `stream` (a torch.cuda.Stream or a raw handle) current for a call on `tensors`.

    Outputs then belong to it, and the tensors are recorded on it: their
    memory is not reused before the call's work is done, even if the caller
    drops them.  The caller orders the stream after the work that makes the inputs."""
    tensors = [t for t in tensors if t is not None]
    device = tensors[0].device
    if device.type != "cuda":
        raise ValueError(f"the operator runs on CUDA tensors, got one on {device}")
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(int(stream), device=device)
    if stream.device != device:
        raise ValueError(f"the stream is on {stream.device}, the tensors on {device}")
    for t in tensors:
        if t.device != device:
            raise ValueError(f"all tensors must be on {device}, got one on {t.device}")
        t.record_stream(stream)
    with torch.cuda.stream(stream):
        yield
