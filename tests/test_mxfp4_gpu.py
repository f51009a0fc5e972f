"""MXFP4 kernels against the format's definition in 64 bits (fp4_ref.py).

The quantizer and its inverse are exact: every code, every scale byte, the
padding and what lies around the outputs are compared bit for bit.
"""

import ctypes

import numpy as np
import pytest
import torch

import MXFP8_quantizer
import fp4_ref
import inputs

pytestmark = pytest.mark.gpu

pkg = MXFP8_quantizer.load_package()
capi = pkg._capi
TORCH = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}


def on_gpu(bits, dtype, ld=None, offset=0):
    """The matrix as a view with row stride ld, `offset` elements into its buffer."""
    m, k = bits.shape
    ld = ld or k
    buf = torch.full((m * ld + offset + 16,), 0x7FC0, dtype=torch.int16, device="cuda")
    view = buf[offset:offset + m * ld].view(m, ld)[:, :k]
    view.copy_(torch.from_numpy(np.ascontiguousarray(bits).view(np.int16)))
    return view.view(TORCH[dtype])


def check_quantize(bits, dtype, **layout):
    q, s = pkg.quantize_mxfp4(on_gpu(bits, dtype, **layout))
    codes, scale = fp4_ref.quantize(bits, dtype)
    np.testing.assert_array_equal(s.cpu().numpy(), fp4_ref.pack_scales(scale))
    np.testing.assert_array_equal(q.cpu().numpy(), fp4_ref.pack_codes(codes))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 32), (1, 4096), (3, 31), (5, 33), (32, 256), (33, 257), (127, 640),
                                 (128, 96), (129, 1000), (300, 8), (1000, 4064), (2, 16384)])
def test_quantize(m, k, dtype):
    check_quantize(inputs.normal(m, k, m * 31 + k, dtype, sigma=3.0), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("ld,offset", [(521, 0), (520, 1), (527, 3), (528, 8), (528, 4), (600, 7)])
def test_quantize_strided_and_offset(ld, offset, dtype):
    check_quantize(inputs.normal(70, 520, 5, dtype), dtype, ld=ld, offset=offset)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_quantize_every_pattern_as_a_value_and_as_the_largest(dtype):
    """All 65536 patterns of the type, each beside itself only and each beside a fixed 1.0; infs and NaNs too."""
    every = np.arange(65536, dtype=np.uint16)
    alone = np.zeros((512, 4096), np.uint16)
    alone[:, 5::32] = every.reshape(512, 128)
    one = np.full((512, 4096), 0x3F80 if dtype == "bf16" else 0x3C00, np.uint16)
    one[:, 5::32] = every.reshape(512, 128)
    check_quantize(alone, dtype)
    check_quantize(one, dtype)


def test_quantize_into_given_buffers_leaves_the_rest():
    bits = inputs.normal(100, 72, 1)
    x = on_gpu(bits, "bf16")
    buf = torch.full((100, 128), 0x5A, dtype=torch.uint8, device="cuda")
    s = torch.full((1024,), 0x5A, dtype=torch.uint8, device="cuda")
    q, s2 = pkg.quantize_mxfp4(x, buf[:, 16:64], s)
    codes, scale = fp4_ref.quantize(bits, "bf16")
    assert q.data_ptr() == buf.data_ptr() + 16 and s2 is s
    np.testing.assert_array_equal(q.cpu().numpy(), fp4_ref.pack_codes(codes))
    assert (buf[:, :16] == 0x5A).all() and (buf[:, 64:] == 0x5A).all() and (s[512:] == 0x5A).all()
    np.testing.assert_array_equal(s[:512].cpu().numpy(), fp4_ref.pack_scales(scale))
    with pytest.raises(ValueError):
        pkg.quantize_mxfp4(x, buf[:, :32])               # too few bytes a row
    with pytest.raises(ValueError):
        pkg.quantize_mxfp4(x, s=s[:256])                 # too few scale bytes
    with pytest.raises(ValueError, match="alignment"):
        pkg.quantize_mxfp4(x, buf[:, 8:56])


def test_transposed_input_is_copied():
    bits = inputs.normal(96, 64, 2)
    q, s = pkg.quantize_mxfp4(on_gpu(bits, "bf16").t())
    codes, scale = fp4_ref.quantize(np.ascontiguousarray(bits.T), "bf16")
    np.testing.assert_array_equal(q.cpu().numpy(), fp4_ref.pack_codes(codes))
    np.testing.assert_array_equal(s.cpu().numpy(), fp4_ref.pack_scales(scale))


def round_once(v, out):
    """f64 -> out, the only rounding (the products are exact in f32 and in f64)."""
    with np.errstate(over="ignore"):
        return torch.from_numpy(v).to(torch.float32).to(TORCH[out])


@pytest.mark.parametrize("out", ["bf16", "fp16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 64), (129, 96), (257, 1056), (64, 4096)])
def test_dequantize(rows, cols, out):
    rng = np.random.default_rng(rows + cols)
    q, s, v = fp4_ref.random_matrix(rng, rows, cols, spread=12)
    got = pkg.dequantize_mxfp4(torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda(), TORCH[out])
    assert torch.equal(got.cpu(), round_once(v, out))


def test_dequantize_every_scale_byte():
    codes = np.tile(np.arange(16, dtype=np.uint8), (256, 2))
    scale = np.arange(256, dtype=np.uint8).reshape(256, 1)
    want = torch.from_numpy(fp4_ref.values(codes, scale)).float()
    got = pkg.dequantize_mxfp4(torch.from_numpy(fp4_ref.pack_codes(codes)).cuda(),
                               torch.from_numpy(fp4_ref.pack_scales(scale)).cuda()).cpu()
    assert torch.equal(got.nan_to_num(nan=1e9), want.nan_to_num(nan=1e9))
    assert got[255].isnan().all() and not got[:255].isnan().any()


@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_dequantize_unaligned_output_rows(out):
    """The C entry writes at any element offset and row stride, and nothing around them."""
    rng = np.random.default_rng(3)
    q, s, v = fp4_ref.random_matrix(rng, 37, 96)
    q, s = torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda()
    buf = torch.full((37 * 101 + 8,), -7.0, dtype=TORCH[out], device="cuda")
    view = buf[3:3 + 37 * 101].view(37, 101)
    capi.fp4_dequantize(q.data_ptr(), 37, 96, 48, s.data_ptr(), s.numel(), view.data_ptr(),
                        pkg._launch.OUT_DTYPES[TORCH[out]], 101, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(view[:, :96].cpu(), round_once(v, out))
    assert (view[:, 96:] == -7).all() and (buf[:3] == -7).all() and (buf[3 + 37 * 101:] == -7).all()


def test_empty():
    q, s = pkg.quantize_mxfp4(torch.empty((0, 64), dtype=torch.bfloat16, device="cuda"))
    assert q.shape == (0, 32) and s.numel() == 0
    q, s = pkg.quantize_mxfp4(torch.empty((4, 0), dtype=torch.bfloat16, device="cuda"))
    assert q.shape == (4, 0)
    assert pkg.dequantize_mxfp4(q, s).shape == (4, 0)


def test_on_another_stream_and_in_a_graph():
    x = torch.randn((200, 512), device="cuda").bfloat16()
    want_q, want_s = pkg.quantize_mxfp4(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for given in (side, side.cuda_stream):
        q, s = pkg.quantize_mxfp4(x, stream=given)
        y = pkg.dequantize_mxfp4(q, s, torch.bfloat16, stream=given)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(q, want_q) and torch.equal(s, want_s)
    assert torch.equal(y, pkg.dequantize_mxfp4(q, s, torch.bfloat16))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, s = pkg.quantize_mxfp4(x)
        y = pkg.dequantize_mxfp4(q, s)
    x.copy_(torch.randn_like(x))
    for _ in range(3):
        graph.replay()
    want_q, want_s = pkg.quantize_mxfp4(x)
    assert torch.equal(q, want_q) and torch.equal(s, want_s)
    assert torch.equal(y, pkg.dequantize_mxfp4(want_q, want_s))
    assert capi.device_status() == 0


def test_checked_build_writes_the_same_bytes():
    """Every store of the checked build lies in its output; narrowed windows show that the guards see these kernels."""
    checked = capi.checked_lib()
    word = ctypes.c_uint32(0)
    stream = torch.cuda.current_stream().cuda_stream
    for m, k, ld in ((100, 520, 523), (129, 72, 72), (1, 33, 40)):
        x = on_gpu(inputs.normal(m, k, m), "bf16", ld=ld)
        q, s = pkg.quantize_mxfp4(x)
        q2, s2 = torch.zeros_like(q), torch.zeros_like(s)
        out = torch.zeros((m, 2 * q.shape[1]), device="cuda")
        for slack, expect in ((0, 0), (64, 16)):
            assert checked.mxfp8_checked_window_slack(slack) == 0
            assert checked.mxfp4_quantize(x.data_ptr(), 0, m, k, ld, q2.data_ptr(), q2.stride(0), s2.data_ptr(),
                                          s2.numel(), stream) == 0
            assert checked.mxfp4_dequantize(q.data_ptr(), m, out.shape[1], q.stride(0), s.data_ptr(), s.numel(),
                                            out.data_ptr(), 2, out.shape[1], stream) == 0
            assert checked.mxfp8_device_status(ctypes.byref(word), 1) == 0
            assert word.value == expect, (m, k, slack)
        assert checked.mxfp8_checked_window_slack(0) == 0
        assert torch.equal(q2, q) and torch.equal(s2, s) and torch.equal(out, pkg.dequantize_mxfp4(q, s))
