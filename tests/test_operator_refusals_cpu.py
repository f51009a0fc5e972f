"""Calls of the 4-bit and cache operators that are refused before a device is
touched, beside those of test_mxfp4_cpu.py and test_cache_cpu.py."""

import pytest
import torch

import MXFP8_quantizer

pkg = MXFP8_quantizer.load_package()


@pytest.mark.parametrize("which", ["first missing", "second missing", "second too small", "second narrower",
                                   "second strided", "first missing and second too small"])
def test_read_refuses_an_output_that_is_not_a_whole_pair(which):
    """Both outputs are written whole, so each is checked, also where the other is missing."""
    cache = pkg.allocate_cache(4, 16, 2, 64, device="cpu")
    table, starts = torch.zeros((3, 4), dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    good = torch.zeros((8, 2, 64))
    pair = {"first missing": (None, good), "second missing": (good, None), "second too small": (good, good[:7]),
            "second narrower": (good, good.half()), "second strided": (good, torch.zeros((8, 2, 128))[:, :, ::2]),
            "first missing and second too small": (None, good[:1].half())}[which]
    with pytest.raises(ValueError, match="out must"):
        pkg.cache_read(cache, table, starts, 8, out=pair)
    with pytest.raises(ValueError, match="CUDA"):                # a whole pair gets as far as the device
        pkg.cache_read(cache, table, starts, 8, out=(good, good.clone()))


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("dtype", [torch.float8_e5m2, torch.float8_e4m3fnuz, torch.float8_e8m0fnu, torch.bool])
def test_cache_refuses_other_8_bit_formats(which, dtype):
    """Their bytes would be read as E4M3."""
    cache = pkg.allocate_cache(4, 16, 2, 64, device="cpu")
    other = cache._replace(**{which: getattr(cache, which).view(torch.uint8).view(dtype)})
    rows, slots = torch.zeros((5, 2, 64), dtype=torch.bfloat16), torch.arange(5)
    table, lengths = torch.zeros((3, 4), dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: pkg.cache_write(other, rows, rows, slots),
                 lambda: pkg.cache_read(other, table, torch.zeros(4, dtype=torch.int32), 8),
                 lambda: pkg.cache_attention(rows[:3], other, table, lengths)):
        with pytest.raises(ValueError, match="e4m3"):
            call()
    for view in (torch.uint8, torch.int8):                       # bytes are taken as they are
        same = cache._replace(**{which: getattr(cache, which).view(view)})
        with pytest.raises(ValueError, match="CUDA"):
            pkg.cache_write(same, rows, rows, slots)


@pytest.mark.parametrize("sizes", [(1, 8192, 1, 64), (1, 16, 65537, 32), (1, 16, 1, 1056), (1, 16, 1, 2048),
                                   (2 ** 28, 16, 1, 32), (2 ** 20, 4096, 2, 32)])
def test_allocate_cache_refuses_what_every_call_would(sizes):
    """Before any memory is taken: these sizes were allocated, and each call on them then refused."""
    with pytest.raises(ValueError, match="a cache needs"):
        pkg.allocate_cache(*sizes, device="meta")


@pytest.mark.parametrize("sizes", [(1, 4096, 1, 32), (1, 1, 65536, 32), (1, 16, 1, 1024), (2 ** 28 - 1, 16, 1, 32), (0, 16, 2, 64)])
def test_allocate_cache_takes_the_limits(sizes):
    cache = pkg.allocate_cache(*sizes, device="meta")
    assert cache.k.shape == (sizes[0], sizes[2], sizes[1], sizes[3])
