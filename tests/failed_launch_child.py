"""Child process for tests/test_failed_launch_gpu.py: calls whose launch the
driver refuses (the default stream, while another stream that it waits for is
being captured), each followed by the same call when it is allowed again.

Prints one JSON line: the refused calls' codes and the following calls' codes.
"""

import ctypes
import json

import numpy as np
from cuda.bindings import runtime as rt

import new_context_child as base


def main():
    base.ok(rt.cudaSetDevice(0))
    lib = base._capi.configure(ctypes.CDLL(str(base._capi.LIB_PATH)))
    bits = np.full((128, 256), 0x3F80, np.uint16)
    x, q, s, y = base.put(bits), base.put(np.zeros(128 * 256, np.uint8)), base.put(np.zeros(4096, np.uint8)), base.put(
        np.zeros(128 * 256 * 4, np.uint8))
    cache = base._capi.Cache(*(base.put(np.zeros(64 * 64, np.uint8)) for _ in range(2)),
                             *(base.put(np.zeros(64 * 2, np.uint8)) for _ in range(2)), 4, 1, 16, 64)
    slots, table, lengths = base.put(np.arange(8)), base.put(np.zeros((1, 1), np.int32)), base.put(np.array([8, 8], np.int32))
    starts = base.put(np.array([0, 8], np.int32))
    need = lib.mxfp8_cache_attention_workspace(cache, 1, 1)
    ws = base.put(np.zeros(need, np.uint8))
    calls = {
        "quantize": lambda: lib.mxfp8_quantize(x, 0, 128, 256, 256, q, 128, 256, 256, s, 4096, None),
        "quantize_noalloc": lambda: lib.mxfp8_quantize_noalloc(x, 0, 128, 256, 256, q, 128, 256, 256, s, 4096, None),
        "quantize into rows at any offset": lambda: lib.mxfp8_quantize(x, 0, 100, 200, 256, q + 1, 100, 224, 224, s, 4096, None),
        "dequantize": lambda: lib.mxfp8_dequantize(q, 128, 256, 256, s, 4096, y, 2, 256, None),
        "mxfp4_quantize": lambda: lib.mxfp4_quantize(x, 0, 128, 256, 256, q, 128, s, 4096, None),
        "mxfp4_dequantize": lambda: lib.mxfp4_dequantize(q, 128, 256, 128, s, 4096, y, 2, 256, None),
        "narrow product": lambda: lib.mxfp4_gemm(q, 1, 128, s, 4096, q, 128, 128, s, 4096, 256, y, 2, 128, None),
        "wide product": lambda: lib.mxfp4_gemm(q, 128, 128, s, 4096, q, 128, 128, s, 4096, 256, y, 2, 128, None),
        "empty product": lambda: lib.mxfp4_gemm(q, 128, 128, s, 4096, q, 128, 128, s, 4096, 0, y, 2, 128, None),
        "cache_write": lambda: lib.mxfp8_cache_write(cache, x, 64, 64, x, 64, 64, 0, 8, slots, None),
        "cache_read": lambda: lib.mxfp8_cache_read(cache, table, 1, 1, 1, starts, 8, y, y + 4096, 0, None),
        "cache_attention": lambda: lib.mxfp8_cache_attention(cache, x, 64, 64, 0, 1, 1, table, 1, 1, lengths, 1.0, y, None,
                                                             ws, need, None),
    }
    stream = base.ok(rt.cudaStreamCreate())                 # one that the default stream waits for
    refused, after = {}, {}
    for call in calls.values():
        assert call() == 0
    for name, call in calls.items():
        base.ok(rt.cudaDeviceSynchronize())
        base.ok(rt.cudaStreamBeginCapture(stream, rt.cudaStreamCaptureMode.cudaStreamCaptureModeRelaxed))
        refused[name] = call()
        rt.cudaStreamEndCapture(stream)                     # invalidated by the call
        rt.cudaGetLastError()                               # of this script's runtime, not the library's
        after[name] = call()
        again = call()
        assert again == 0, (name, again)
    base.ok(rt.cudaDeviceSynchronize())
    print(json.dumps({"refused": refused, "after": after}), flush=True)


if __name__ == "__main__":
    main()
