"""Child process for tests/test_new_context_gpu.py: the library's calls in the
primary context, in a second context of the same device, and in the primary one
again.

Runs without torch, so that only this script and the library touch CUDA.
Prints one JSON line: per context, the calls' status codes and whether each
output has the bytes it had in the first.
"""

import ctypes
import json
import pathlib
import sys

import numpy as np
from cuda.bindings import driver as drv
from cuda.bindings import runtime as rt

ROOT = pathlib.Path(__file__).resolve().parent.parent
sys.path.insert(0, str(ROOT / "mxfp8-quantizer_b200"))
import _capi  # noqa: E402  (ctypes binding only: it imports nothing else of the package)


def ok(res):
    err, *vals = res
    if int(err) != 0:
        raise SystemExit(f"CUDA call failed: {err}")
    return vals[0] if len(vals) == 1 else tuple(vals)


def put(a):
    p = int(ok(rt.cudaMalloc(max(a.nbytes, 16))))
    ok(rt.cudaMemcpy(p, a.ctypes.data, a.nbytes, rt.cudaMemcpyKind.cudaMemcpyHostToDevice))
    return p


def get(p, n):
    a = np.empty(n, np.uint8)
    ok(rt.cudaMemcpy(a.ctypes.data, p, n, rt.cudaMemcpyKind.cudaMemcpyDeviceToHost))
    return a


def calls(lib):
    """Each kind of kernel once: [(status code, output bytes or None)]."""
    rng = np.random.default_rng(0)
    out = []

    def note(rc, p, n):
        out.append((rc, get(p, n) if rc == 0 else None))

    # quantizers: rows on 16 bytes, rows off them; without allocation; 4 bits
    for ld in (1024, 1025):
        bits = (rng.standard_normal((256, ld)).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
        x, q, s = put(bits), put(np.zeros(256 * 1024, np.uint8)), put(np.zeros(256 * 32, np.uint8))
        for entry in (lib.mxfp8_quantize, lib.mxfp8_quantize_noalloc):
            note(entry(x, 0, 256, 1024, ld, q, 256, 1024, 1024, s, 256 * 32, None), q, 256 * 1024)
    note(lib.mxfp4_quantize(x, 0, 256, 1024, 1025, q, 512, s, 256 * 32, None), q, 256 * 512)
    # the product's forms: narrow of every width (one split over a cluster), wide, wide with columns as rows
    k = 512
    a_q, a_s = put(rng.integers(0, 256, (4096, k // 2), np.uint8)), put(np.full(4096 * k // 32, 127, np.uint8))
    c = put(np.zeros(4096 * 2048 * 4, np.uint8))
    for m, n, ld in ((1, 128, 128), (32, 128, 128), (64, 128, 128), (128, 128, 128), (2048, 2048, 2048), (4096, 1300, 1301)):
        rc = lib.mxfp4_gemm(a_q, m, k // 2, a_s, 4096 * k // 32, a_q, n, k // 2, a_s, 4096 * k // 32, k, c, 0, ld, None)
        note(rc, c, 2 * ld * m)
    # attention, each width and both row counts
    for dim, group in ((64, 1), (64, 16), (128, 1), (128, 16), (192, 4), (256, 8)):
        rows = 4 * 16
        cache = _capi.Cache(*(put(rng.integers(0, 120, rows * dim, np.uint8)) for _ in range(2)),
                            *(put(np.full(rows * dim // 32, 120, np.uint8)) for _ in range(2)), 4, 1, 16, dim)
        q = put(rng.integers(0, 0x3C00, 2 * group * dim).astype(np.uint16))
        table, lengths = put(np.array([[0, 1], [2, 3]], np.int32)), put(np.array([32, 20], np.int32))
        need = lib.mxfp8_cache_attention_workspace(cache, 2, group)
        o, ws = put(np.zeros(2 * group * dim * 2, np.uint8)), int(ok(rt.cudaMalloc(need)))
        rc = lib.mxfp8_cache_attention(cache, q, group * dim, dim, 1, 2, group, table, 2, 2, lengths, dim ** -0.5, o, None,
                                       ws, need, None)
        note(rc, o, 2 * group * dim * 2)
    word = ctypes.c_uint32(1)
    out.append((lib.mxfp8_device_status(ctypes.byref(word), 0), np.array([word.value])))
    return out


def main():
    ok(drv.cuInit(0))
    dev = ok(drv.cuDeviceGet(0))
    primary = ok(drv.cuDevicePrimaryCtxRetain(dev))
    ok(drv.cuCtxSetCurrent(primary))
    lib = _capi.configure(ctypes.CDLL(str(_capi.LIB_PATH)))
    first = calls(lib)
    try:
        other = ok(drv.cuCtxCreate(0, dev))
    except TypeError:  # newer bindings take creation parameters first
        other = ok(drv.cuCtxCreate(None, 0, dev))
    ok(drv.cuCtxSetCurrent(other))
    second = calls(lib)
    ok(drv.cuCtxSetCurrent(primary))
    third = calls(lib)
    print(json.dumps({"codes": [[rc for rc, _ in t] for t in (first, second, third)],
                      "same": [[a is not None and b is not None and bool((a == b).all())
                                for (_, a), (_, b) in zip(first, t)] for t in (second, third)],
                      "some": [bool(a.any()) for _, a in first[:-1] if a is not None]}), flush=True)


if __name__ == "__main__":
    main()
