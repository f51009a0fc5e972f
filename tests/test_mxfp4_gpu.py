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
CODES = {"bf16": capi.BF16, "fp16": capi.FP16, "f32": capi.F32}


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
                        CODES[out], 101, torch.cuda.current_stream().cuda_stream)
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


# --------------------------------------------------------------------------
# the product
# --------------------------------------------------------------------------

HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "f32": 2.0 ** -24}


def check_gemm(m, n, k, out, seed=0, spread=3):
    """Against 64 bits.  The products are exact; each of the at most k f32
    additions of an output is off by at most one unit in the last place
    (2^-23) of a partial sum, which is at most sum |a||b|; then one rounding."""
    rng = np.random.default_rng(seed + m * 7 + n * 3 + k)
    a_q, a_s, a = fp4_ref.random_matrix(rng, m, k, spread)
    b_q, b_s, b = fp4_ref.random_matrix(rng, n, k, spread)
    a_q, a_s, b_q, b_s = (torch.from_numpy(t).cuda() for t in (a_q, a_s, b_q, b_s))
    got = pkg.mxfp4_gemm(a_q, b_q, a_s, b_s, TORCH[out])
    assert capi.device_status(clear=True) == 0
    a, b = torch.from_numpy(a).cuda(), torch.from_numpy(b).cuda()
    want = a @ b.t()
    room = k * 2.0 ** -23 * (a.abs() @ b.abs().t()) + HALF_STEP[out] * want.abs() * (1 + 2.0 ** -8)
    off = (got.double() - want).abs() - room
    assert not (off > 0).any(), (m, n, k, out, off.max().item(), (off > 0).sum().item())
    return got


@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (1, 128, 64), (1, 128, 256), (1, 4096, 4096), (16, 300, 96),
                                   (17, 129, 160), (32, 256, 1024), (33, 100, 352), (64, 512, 2048), (65, 17, 64),
                                   (77, 1000, 2080), (128, 128, 128), (129, 255, 288), (200, 1024, 4096),
                                   (300, 77, 1056)])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_gemm(m, n, k, out):
    check_gemm(m, n, k, out)


@pytest.mark.parametrize("m,n,k,out", [(4096, 1280, 512, "fp16"), (4096, 1280, 96, "f32"), (2048, 2304, 288, "bf16"),
                                       (4000, 1296, 544, "bf16"), (4095, 1301, 256, "fp16"), (2500, 2500, 1024, "f32"),
                                       (10000, 520, 320, "bf16"), (2600, 1024, 2080, "bf16"), (2600, 1000, 4096, "f32"),
                                       (300, 10000, 160, "fp16"), (700, 4096, 2048, "bf16")])
def test_gemm_many_tiles(m, n, k, out):
    check_gemm(m, n, k, out)


@pytest.mark.parametrize("m,n,k", [(65, 129, 32), (300, 515, 512), (513, 1001, 96), (256, 257, 4096), (1025, 2047, 288),
                                   (3001, 2999, 160)])
@pytest.mark.parametrize("out", ["bf16", "fp16", "f32"])
def test_gemm_rows_off_32_bytes(m, n, k, out):
    check_gemm(m, n, k, out, seed=1)


@pytest.mark.parametrize("m", [1, 16, 40, 130, 4096])
def test_gemm_small_integers_are_exact(m):
    """All scales 1 and k <= 1024: every partial sum is a multiple of 1/4 below 2^16, so f32 holds it."""
    rng = np.random.default_rng(m)
    scale = np.full((m, 32), 127, np.uint8)
    codes = rng.integers(0, 16, (m, 1024)).astype(np.uint8)
    b_codes = rng.integers(0, 16, (1280, 1024)).astype(np.uint8)
    b_scale = np.full((1280, 32), 127, np.uint8)
    t = [torch.from_numpy(x).cuda() for x in (fp4_ref.pack_codes(codes), fp4_ref.pack_codes(b_codes),
                                              fp4_ref.pack_scales(scale), fp4_ref.pack_scales(b_scale))]
    want = torch.from_numpy(fp4_ref.values(codes, scale)).cuda() @ torch.from_numpy(fp4_ref.values(b_codes, b_scale)).cuda().t()
    assert torch.equal(pkg.mxfp4_gemm(*t).double(), want)


@pytest.mark.parametrize("m,n,ld,offset", [(5, 100, 101, 3), (70, 130, 137, 1), (2000, 2560, 2561, 5)])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_gemm_into_any_row_stride(m, n, ld, offset, out):
    buf = torch.full((m * ld + offset + 8,), -7.0, dtype=TORCH[out], device="cuda")
    view = buf[offset:offset + m * ld].view(m, ld)[:, :n]
    got = check_gemm(m, n, 96, out)
    rng = np.random.default_rng(m * 7 + n * 3 + 96)
    a_q, a_s, _ = fp4_ref.random_matrix(rng, m, 96, 3)
    b_q, b_s, _ = fp4_ref.random_matrix(rng, n, 96, 3)
    a_q, a_s, b_q, b_s = (torch.from_numpy(t).cuda() for t in (a_q, a_s, b_q, b_s))
    assert pkg.mxfp4_gemm(a_q, b_q, a_s, b_s, out=view) is view
    room = 96 * 2.0 ** -22 * 36 * 64 * 96 + 2 * HALF_STEP[out] * got.double().abs()   # two orders of one sum
    assert ((view.double() - got.double()).abs() <= room).all()
    rest = buf.clone()
    rest[offset:offset + m * ld].view(m, ld)[:, :n] = -7.0
    assert (rest == -7.0).all()


def test_gemm_padded_rows_and_views():
    """Operands that are column and row slices of larger matrices."""
    rng = np.random.default_rng(11)
    a_q, a_s, a = fp4_ref.random_matrix(rng, 30, 64)
    b_q, b_s, b = fp4_ref.random_matrix(rng, 90, 64)
    big_a = torch.full((30, 80), 0xFF, dtype=torch.uint8, device="cuda")
    big_b = torch.full((128, 64), 0xFF, dtype=torch.uint8, device="cuda")
    va, vb = big_a[:, 16:48], big_b[20:110, 32:]
    va.copy_(torch.from_numpy(a_q)), vb.copy_(torch.from_numpy(b_q))
    got = pkg.mxfp4_gemm(va, vb, torch.from_numpy(a_s).cuda(), torch.from_numpy(b_s).cuda())
    want = pkg.mxfp4_gemm(torch.from_numpy(a_q).cuda(), torch.from_numpy(b_q).cuda(), torch.from_numpy(a_s).cuda(),
                          torch.from_numpy(b_s).cuda())
    assert torch.equal(got, want)


@pytest.mark.parametrize("m,n", [(3, 200), (150, 200), (2560, 2048)])
def test_gemm_nan_blocks_reach_their_outputs_only(m, n):
    rng = np.random.default_rng(m)
    k = 256
    a_codes, b_codes = (rng.integers(0, 16, (r, k)).astype(np.uint8) for r in (m, n))
    a_scale, b_scale = (np.full((r, k // 32), 127, np.uint8) for r in (m, n))
    a_scale[m - 1, 3] = 255
    b_scale[5, 0] = 255
    t = [torch.from_numpy(x).cuda() for x in (fp4_ref.pack_codes(a_codes), fp4_ref.pack_codes(b_codes),
                                              fp4_ref.pack_scales(a_scale), fp4_ref.pack_scales(b_scale))]
    got = pkg.mxfp4_gemm(*t)
    nan = torch.zeros((m, n), dtype=torch.bool, device="cuda")
    nan[m - 1] = True
    nan[:, 5] = True
    assert torch.equal(got.isnan(), nan)


def test_gemm_extreme_scales():
    """Scales at both ends of their range: 2^-127 * 2^127 products are ordinary numbers."""
    codes = np.full((4, 64), 2, np.uint8)                 # 1.0
    low, high = np.full((4, 2), 0, np.uint8), np.full((4, 2), 254, np.uint8)
    q = torch.from_numpy(fp4_ref.pack_codes(codes)).cuda()
    s_low, s_high = (torch.from_numpy(fp4_ref.pack_scales(s)).cuda() for s in (low, high))
    assert (pkg.mxfp4_gemm(q, q, s_low, s_high) == 64.0).all()


def test_gemm_empty():
    z = torch.empty((0, 32), dtype=torch.uint8, device="cuda")
    none = torch.empty(0, dtype=torch.uint8, device="cuda")
    q, s = torch.zeros((4, 32), dtype=torch.uint8, device="cuda"), torch.zeros(512, dtype=torch.uint8, device="cuda")
    assert pkg.mxfp4_gemm(z, q, none, s).shape == (0, 4)
    assert pkg.mxfp4_gemm(q, z, s, none).shape == (4, 0)
    assert (pkg.mxfp4_gemm(q[:, :0], q[:, :0], none, none) == 0).all()


@pytest.mark.parametrize("m", [2, 100, 3000])
def test_gemm_repeats_bit_for_bit_on_streams_and_in_graphs(m):
    rng = np.random.default_rng(m)
    sets = []
    for i in range(2):
        a_q, a_s, _ = fp4_ref.random_matrix(rng, m, 2048)
        b_q, b_s, _ = fp4_ref.random_matrix(rng, 2048, 2048)
        sets.append([torch.from_numpy(x).cuda() for x in (a_q, b_q, a_s, b_s)])
    want = [pkg.mxfp4_gemm(*t) for t in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = [pkg.mxfp4_gemm(*t, stream=side) for t in sets]
    here = [pkg.mxfp4_gemm(*t) for t in sets]            # at the same time as the side stream's
    torch.cuda.current_stream().wait_stream(side)
    for w, o, h in zip(want, other, here):
        assert torch.equal(w, o) and torch.equal(w, h)
    graph = torch.cuda.CUDAGraph()
    static = [t.clone() for t in sets[0]]
    with torch.cuda.graph(graph):
        c = pkg.mxfp4_gemm(*static)
        c2 = pkg.mxfp4_gemm(*sets[1])
    for t, w in zip((sets[1], sets[0]), (want[1], want[0])):
        for dst, src in zip(static, t):
            dst.copy_(src)
        graph.replay()
        assert torch.equal(c, w) and torch.equal(c2, want[1])
    assert capi.device_status() == 0


def test_quantize_then_product():
    """x W^T through quantize_mxfp4 and mxfp4_gemm equals the product of the dequantized matrices."""
    x = torch.randn((70, 500), device="cuda").bfloat16()
    w = torch.randn((300, 500), device="cuda").bfloat16()
    (xq, xs), (wq, ws) = pkg.quantize_mxfp4(x), pkg.quantize_mxfp4(w)
    got = pkg.mxfp4_gemm(xq, wq, xs, ws)
    a, b = (pkg.dequantize_mxfp4(*t).double() for t in ((xq, xs), (wq, ws)))
    room = 512 * 2.0 ** -23 * (a.abs() @ b.abs().t())
    assert ((got.double() - a @ b.t()).abs() <= room).all()


def test_gemm_checked_build():
    """The checked build's guards see every store of the product."""
    checked = capi.checked_lib()
    word = ctypes.c_uint32(0)
    rng = np.random.default_rng(2)
    for m, n, k in ((3, 100, 64), (77, 130, 2080), (2560, 2056, 96), (2560, 2051, 96)):
        a_q, a_s, _ = fp4_ref.random_matrix(rng, m, k)
        b_q, b_s, _ = fp4_ref.random_matrix(rng, n, k)
        a_q, a_s, b_q, b_s = (torch.from_numpy(t).cuda() for t in (a_q, a_s, b_q, b_s))
        want = pkg.mxfp4_gemm(a_q, b_q, a_s, b_s)
        out = torch.zeros_like(want)
        for slack, expect in ((0, 0), (4, 16)):
            assert checked.mxfp8_checked_window_slack(slack) == 0
            assert checked.mxfp4_gemm(a_q.data_ptr(), m, k // 2, a_s.data_ptr(), a_s.numel(), b_q.data_ptr(), n, k // 2,
                                      b_s.data_ptr(), b_s.numel(), k, out.data_ptr(), 2, n,
                                      torch.cuda.current_stream().cuda_stream) == 0
            assert checked.mxfp8_device_status(ctypes.byref(word), 1) == 0
            assert word.value == expect
        assert checked.mxfp8_checked_window_slack(0) == 0
        assert torch.equal(out, want)
