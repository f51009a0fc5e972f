"""Capturing the 4-bit and cache operators in a process that has not run those
kernels before: only the device's status word has to be there (any call before)."""

import pathlib
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = pathlib.Path(__file__).resolve().parent.parent

CHILD = """
import torch
import MXFP8_quantizer

pkg = MXFP8_quantizer.load_package()
pkg._capi.device_status()
x = torch.randn((40, 512), device="cuda").half()
w = torch.randn((384, 512), device="cuda").half()
cache = pkg.allocate_cache(8, 16, 2, 64)
slots = torch.arange(40, device="cuda")
table = torch.tensor([[0, 1, 2], [1, 2, 0]], dtype=torch.int32, device="cuda")
lengths = torch.tensor([40, 17], dtype=torch.int32, device="cuda")
starts = torch.tensor([0, 40, 57], dtype=torch.int32, device="cuda")


def step():
    xq, xs = pkg.quantize_mxfp4(x)
    wq, ws = pkg.quantize_mxfp4(w)
    y = pkg.mxfp4_gemm(xq, wq, xs, ws, torch.float16)
    k, v = y[:, :128].view(40, 2, 64), y[:, 128:256].view(40, 2, 64)
    pkg.cache_write(cache, k, v, slots)
    q = y[:2, 128:].reshape(2, 4, 64)
    rows = pkg.cache_read(cache, table, starts, 57, torch.float16)
    return y, pkg.dequantize_mxfp4(xq, xs, torch.float16), *rows, pkg.cache_attention(q, cache, table, lengths)


graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = step()
for _ in range(2):
    x.normal_()
    graph.replay()
    got = [t.clone() for t in captured]
    for a, b in zip(got, step()):
        assert torch.equal(a, b)
assert pkg._capi.device_status() == 0
print("captured")
"""


def test_first_use_of_every_kernel_inside_a_capture():
    done = subprocess.run([sys.executable, "-c", CHILD], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]
