"""MXFP4 matrices of a single row, whose row stride means nothing: any is taken."""

import numpy as np
import pytest
import torch

import fp4_ref
from test_mxfp4_gpu import capi, pkg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("stride", [1, 40, 129, 512])
def test_any_stride_of_one_row(stride):
    rng = np.random.default_rng(stride)
    q, s, v = fp4_ref.random_matrix(rng, 1, 256)
    b_q, b_s, b = (torch.from_numpy(t).cuda() for t in fp4_ref.random_matrix(rng, 200, 256))
    q, s = torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda()
    row = torch.as_strided(q, (1, 128), (stride, 1))
    assert torch.equal(pkg.dequantize_mxfp4(row, s), pkg.dequantize_mxfp4(q, s))
    want = pkg.mxfp4_gemm(q, b_q, s, b_s)
    assert torch.equal(pkg.mxfp4_gemm(row, b_q, s, b_s), want)
    assert torch.equal(pkg.mxfp4_gemm(b_q, row, b_s, s), pkg.mxfp4_gemm(b_q, q, b_s, s))
    out = torch.as_strided(torch.empty(200, device="cuda"), (1, 200), (stride, 1))
    assert torch.equal(pkg.mxfp4_gemm(q, b_q, s, b_s, out=out), want)
    x = torch.randn(1, 200, device="cuda").bfloat16()
    want_q, want_s = pkg.quantize_mxfp4(x)
    into = torch.as_strided(torch.zeros(112, dtype=torch.uint8, device="cuda"), (1, 112), (stride, 1))
    got_q, got_s = pkg.quantize_mxfp4(torch.as_strided(x, (1, 200), (stride, 1)), into)
    assert torch.equal(got_q, want_q) and torch.equal(got_s, want_s)
    assert capi.device_status() == 0
