"""The 4-bit and cache operators called from two host threads at once, each on a
stream of its own, and on the default stream by its raw handle."""

import pathlib
import sys
import threading

import pytest
import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent))
import MXFP8_quantizer

pytestmark = pytest.mark.gpu

pkg = MXFP8_quantizer.load_package()


class Step:
    """A projection in 4 bits, its K and V into the cache, attention over it, and the rows read back."""

    def __init__(self, seed, tokens, n):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.x = torch.randn((tokens, 512), device="cuda", generator=g).half()
        self.w = torch.randn((512, 512), device="cuda", generator=g).half()
        self.cache = pkg.allocate_cache(64, 16, 2, 64)
        self.slots = torch.arange(tokens, device="cuda")
        self.table = torch.arange(64, dtype=torch.int32, device="cuda").view(1, 64).repeat(n, 1)
        self.lengths = (torch.arange(n, device="cuda") * 41 % tokens).int()
        self.starts = torch.arange(n + 1, dtype=torch.int32, device="cuda") * 5
        self.n = n

    def run(self, **stream):
        x = pkg.quantize_mxfp4(self.x, **stream)
        w = pkg.quantize_mxfp4(self.w, **stream)
        y = pkg.mxfp4_gemm(x[0], w[0], x[1], w[1], torch.float16, **stream)
        back = pkg.dequantize_mxfp4(*x, torch.float16, **stream)
        rows = (y.shape[0], 2, 64)
        pkg.cache_write(self.cache, y[:, :128].unflatten(1, rows[1:]), y[:, 128:256].unflatten(1, rows[1:]), self.slots,
                        **stream)
        q = y[:self.n, 256:].unflatten(1, (4, 64))
        return (y, back, *pkg.cache_read(self.cache, self.table, self.starts, 5 * self.n, torch.float16, **stream),
                *pkg.cache_attention(q, self.cache, self.table, self.lengths, return_lse=True, **stream))


def test_two_threads_on_two_streams():
    steps = [Step(1, 600, 37), Step(2, 301, 5)]
    want = [[t.clone() for t in s.run()] for s in steps]
    torch.cuda.synchronize()
    got, failed = [None, None], []
    ready = threading.Barrier(2)

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                ready.wait(60)
                kept = [steps[i].run() for _ in range(30)]
                stream.synchronize()
            got[i] = kept
        except Exception as e:  # the thread's failure is the test's
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not failed, failed
    for i in range(2):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i]))
    assert pkg._capi.device_status() == 0


def test_the_default_stream_by_its_handle():
    step = Step(3, 100, 3)
    want = step.run()
    assert torch.cuda.default_stream().cuda_stream == 0
    got = step.run(stream=0)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
