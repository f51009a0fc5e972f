"""MXFP4 without a GPU: the binding covers its header, and bad arguments are
refused before a device is touched."""

import pathlib
import re

import numpy as np
import pytest
import torch

import MXFP8_quantizer
import fp4_ref

ROOT = pathlib.Path(__file__).resolve().parent.parent
pkg = MXFP8_quantizer.load_package()
capi = pkg._capi


def test_header_binding_and_libraries_agree():
    text = (ROOT / "include" / "mxfp4.h").read_text()
    declared = sorted(set(re.findall(r"MXFP8_API\s+[\w\s\*]+?\b(mxfp4_\w+)\s*\(", text)))
    assert declared == sorted(capi.FP4_EXPORTS)
    for name in declared:
        assert hasattr(capi.lib(), name) and hasattr(capi.checked_lib(), name), name


@pytest.mark.parametrize("change,match", [
    (dict(dtype=2), "dtype"),
    (dict(m=-1), "sizes"),
    (dict(k=2 ** 31), "sizes"),
    (dict(ld_x=99), "sizes"),
    (dict(ld_q=48), "sizes"),            # 100 columns pad to 128: 64 bytes
    (dict(ld_q=72), "alignment"),
    (dict(x=0), "NULL"),
    (dict(q=0), "NULL"),
    (dict(s=0), "NULL"),
    (dict(x=0x1001), "alignment"),
    (dict(q=0x2008), "alignment"),
    (dict(s=0x3004), "alignment"),
    (dict(s_bytes=511), "scale buffer"),
])
def test_quantize_refuses(change, match):
    a = dict(x=0x1000, dtype=0, m=16, k=100, ld_x=100, q=0x2000, ld_q=64, s=0x3000, s_bytes=512)
    a.update(change)
    with pytest.raises(ValueError, match=match):
        capi.fp4_quantize(*a.values(), 0)


@pytest.mark.parametrize("change,match", [
    (dict(code=9), "dtype"),
    (dict(cols=48), "sizes"),
    (dict(ld_q=48), "sizes"),
    (dict(ld_out=100), "sizes"),
    (dict(out=0), "NULL"),
    (dict(out=0x4001), "alignment"),
    (dict(q=0x2001), "alignment"),
    (dict(s_bytes=511), "scale buffer"),
])
def test_dequantize_refuses(change, match):
    a = dict(q=0x2000, rows=16, cols=128, ld_q=64, s=0x3000, s_bytes=512, out=0x4000, code=0, ld_out=128)
    a.update(change)
    with pytest.raises(ValueError, match=match):
        capi.fp4_dequantize(*a.values(), 0)


def test_empty_matrices_are_no_ops():
    capi.fp4_quantize(0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    capi.fp4_quantize(0, 0, 0, 64, 64, 0, 32, 0, 0, 0)
    capi.fp4_dequantize(0, 0, 32, 16, 0, 0, 0, 0, 32, 0)


def test_wrappers_refuse_wrong_tensors():
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    q, s = torch.zeros((4, 32), dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.quantize_mxfp4(x)
    with pytest.raises(ValueError, match="2-D"):
        pkg.quantize_mxfp4(x[0])
    with pytest.raises(ValueError, match="bfloat16"):
        pkg.quantize_mxfp4(x.float())
    with pytest.raises(ValueError, match="CUDA"):
        pkg.dequantize_mxfp4(q, s)
    with pytest.raises(ValueError, match="32 columns"):
        pkg.dequantize_mxfp4(q[:, :24], s)
    with pytest.raises(ValueError, match="row-major"):
        pkg.dequantize_mxfp4(q.t(), s)
    with pytest.raises(ValueError, match="row-major"):
        pkg.dequantize_mxfp4(q.view(torch.float8_e4m3fn), s)
    with pytest.raises(ValueError, match="out_dtype"):
        pkg.dequantize_mxfp4(q, s, torch.float64)


def test_the_64_bit_form_rounds_to_nearest_even():
    """Each midpoint goes to its even neighbour, each scale border to the smaller scale."""
    x = np.zeros((2, 32), np.float32)
    x[0, :9] = [6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25]
    x[1, :2] = [6.03125, 0.5]                       # the next bf16 above 6: the scale doubles
    bits = (x.view(np.uint32) >> 16).astype(np.uint16)
    codes, scale = fp4_ref.quantize(bits, "bf16")
    assert codes[0, :9].tolist() == [7, 0, 2, 2, 4, 4, 6, 6, 8]
    assert scale.tolist() == [[127], [128]] and codes[1, :2].tolist() == [5, 0]


@pytest.mark.parametrize("change,match", [
    (dict(code=9), "dtype"),
    (dict(k=48), "sizes"),
    (dict(ld_a=48), "sizes"),
    (dict(ld_out=7), "sizes"),
    (dict(out=0), "NULL"),
    (dict(out=0x7002), "alignment"),
    (dict(a=0), "NULL"),
    (dict(b_s=0), "NULL"),
    (dict(a=0x1008), "alignment"),
    (dict(ld_b=72), "alignment"),
    (dict(b_s=0x4004), "alignment"),
    (dict(a_s_bytes=511), "scale buffer"),
    (dict(b_s_bytes=511), "scale buffer"),
])
def test_gemm_refuses(change, match):
    a = dict(a=0x1000, m=4, ld_a=64, a_s=0x2000, a_s_bytes=512, b=0x3000, n=8, ld_b=64, b_s=0x4000, b_s_bytes=512,
             k=128, out=0x7000, code=2, ld_out=8)
    a.update(change)
    with pytest.raises(ValueError, match=match):
        capi.fp4_gemm(*a.values(), 0)


def test_gemm_wrapper_refuses():
    q, s = torch.zeros((4, 32), dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.mxfp4_gemm(q, q, s, s)
    with pytest.raises(ValueError, match="same number of columns"):
        pkg.mxfp4_gemm(q, q[:, :16], s, s)
    with pytest.raises(ValueError, match="out must"):
        pkg.mxfp4_gemm(q, q, s, s, out=torch.zeros((4, 5)))
    with pytest.raises(ValueError, match="out_dtype"):
        pkg.mxfp4_gemm(q, q, s, s, torch.float64)
    with pytest.raises(ValueError, match="contiguous"):
        pkg.mxfp4_gemm(q, q, s[::2], s)
