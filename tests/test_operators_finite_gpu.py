"""The product and the attention over the cases of their own tests, with a check
that a NaN does not pass, and with each element's own room."""

import math

import numpy as np
import pytest
import torch

import fp4_ref
from strict import assert_within
from test_cache_gpu import LENGTHS, attention_case, capi, pkg, rows_of
from test_cache_ranges_gpu import check_elements
from test_mxfp4_gpu import HALF_STEP, TORCH

pytestmark = pytest.mark.gpu


def operands(m, n, k, seed, spread=3):
    rng = np.random.default_rng(seed)
    sides = []
    for rows in (m, n):
        q, s, v = fp4_ref.random_matrix(rng, rows, k, spread)
        sides.append((torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda(), torch.from_numpy(v).cuda()))
    return sides


def product_room(a, b, want, out):
    """k additions of exact products, each off by one unit in the last place (2^-23) of a partial sum that is at most
    sum |a||b|; then one rounding (which of a value that room off)."""
    room = a.shape[1] * 2.0 ** -23 * (a.abs() @ b.abs().t())
    return room + HALF_STEP[out] * (want.abs() + room)


@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (1, 128, 256), (1, 4096, 4096), (16, 300, 96), (17, 129, 160), (33, 100, 352),
                                   (64, 512, 2048), (65, 17, 64), (77, 1000, 2080), (129, 255, 288), (200, 1024, 4096),
                                   (256, 257, 4096), (513, 1001, 96), (700, 4096, 2048), (2600, 1000, 4096),
                                   (4095, 1301, 256), (10000, 520, 320), (3001, 2999, 160)])
@pytest.mark.parametrize("out", ["bf16", "fp16", "f32"])
def test_product(m, n, k, out):
    (a_q, a_s, a), (b_q, b_s, b) = operands(m, n, k, m + n + k)
    want = a @ b.t()
    # an output that the call did not write would show
    got = torch.full((m, n), math.nan, dtype=TORCH[out], device="cuda")
    pkg.mxfp4_gemm(a_q, b_q, a_s, b_s, out=got)
    assert_within(got, want, product_room(a, b, want, out), (m, n, k, out))
    assert capi.device_status(clear=True) == 0


@pytest.mark.parametrize("m,n,ld,offset", [(5, 100, 101, 3), (70, 130, 137, 1), (2000, 2560, 2561, 5), (2000, 2560, 2576, 16)])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_product_into_any_row_stride(m, n, ld, offset, out):
    (a_q, a_s, a), (b_q, b_s, b) = operands(m, n, 96, m)
    buf = torch.full((m * ld + offset + 8,), math.nan, dtype=TORCH[out], device="cuda")
    view = buf[offset:offset + m * ld].view(m, ld)[:, :n]
    pkg.mxfp4_gemm(a_q, b_q, a_s, b_s, out=view)
    want = a @ b.t()
    assert_within(view, want, product_room(a, b, want, out), (m, n, ld))
    view.fill_(math.nan)
    assert buf.isnan().all()                                   # nothing else was written


@pytest.mark.parametrize("heads,group,dim,page,dtype", [(1, 1, 64, 2, "bf16"), (2, 4, 64, 16, "fp16"), (3, 8, 128, 16, "bf16"),
                                                        (1, 16, 128, 64, "fp16"), (2, 5, 192, 8, "bf16"),
                                                        (1, 7, 256, 32, "fp16"), (2, 12, 64, 8, "bf16"),
                                                        (1, 24, 128, 16, "fp16"), (1, 17, 256, 128, "bf16")])
def test_attention(heads, group, dim, page, dtype):
    lengths = [n for n in LENGTHS if n]
    q, cache, table = attention_case(lengths, page, heads, group, dim, dtype, seed=group + dim)
    check_elements(q, cache, table, lengths, page)


@pytest.mark.parametrize("lengths,heads,group,dim", [([20000], 2, 4, 128), ([5000, 1, 9001], 1, 8, 256), ([64] * 300, 2, 2, 64),
                                                     ([1] * 700, 1, 4, 64), ([30000] + [3] * 300, 1, 4, 64)])
def test_attention_splits(lengths, heads, group, dim):
    q, cache, table = attention_case(lengths, 16, heads, group, dim, "bf16", seed=len(lengths))
    check_elements(q, cache, table, lengths, 16)


def test_attention_of_empty_sequences_beside_others():
    lengths = [0, 40, 0, 0, 1000, 0]
    q, cache, table = attention_case(lengths, 16, 2, 4, 128, "fp16", seed=6)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out, lse = pkg.cache_attention(q, cache, table, lens, return_lse=True)
    empty = lens == 0
    assert (out[empty] == 0).all() and (lse[empty] == -math.inf).all()
    assert out.isfinite().all() and lse[~empty].isfinite().all()
    keep = (~empty).nonzero()[:, 0]
    alone = check_elements(q[keep], cache, table[keep], [40, 1000], 16)
    for b, n in ((1, 40), (4, 1000)):                          # whatever is beside them
        k = rows_of(cache.k, cache.k_scales, table, b, n, 16)
        assert k.isfinite().all()
    assert (out[keep].double() - alone.double()).abs().max() <= 2 * 2.0 ** -11 * alone.double().abs().max()


def test_a_decode_step_of_a_layer():
    """Projection in 4 bits, cache write, attention over what was written, step by step: every output a number."""
    batch, heads, group, dim, page, width = 3, 2, 4, 128, 16, 256
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((batch, width), device="cuda", generator=g).bfloat16()
    w = (torch.randn(((heads * group + 2 * heads) * dim, width), device="cuda", generator=g) / 16).bfloat16()
    w_q, w_s = pkg.quantize_mxfp4(w)
    cache = pkg.allocate_cache(8, page, heads, dim)
    table = torch.tensor([[4, 1], [2, 0], [7, 3]], dtype=torch.int32, device="cuda")
    for step in range(20):
        x_q, x_s = pkg.quantize_mxfp4(x)
        y = pkg.mxfp4_gemm(x_q, w_q, x_s, w_s, torch.bfloat16)
        q, k, v = y.split([heads * group * dim, heads * dim, heads * dim], 1)
        pkg.cache_write(cache, k.view(batch, heads, dim), v.view(batch, heads, dim),
                        table[:, step // page].long() * page + step % page)
        out = check_elements(q.view(batch, heads * group, dim), cache, table, [step + 1] * batch, page)
        x = out.reshape(batch, -1)[:, :width] + x * 0.5
    assert capi.device_status() == 0


def test_attention_of_several_tokens_a_sequence():
    """Drafted tokens as rows of one batch: a sequence's table row repeated, the lengths rising by one."""
    page, tokens = 16, 5
    q, cache, table = attention_case([37, 300], page, 2, 4, 128, "bf16", seed=21)
    g = torch.Generator(device="cuda").manual_seed(22)
    q = torch.randn((2 * tokens, 8, 128), device="cuda", generator=g).bfloat16()
    rows = table.repeat_interleave(tokens, 0)
    check_elements(q, cache, rows, [33 + t for t in range(tokens)] + [296 + t for t in range(tokens)], page)
    one = table[:1].expand(tokens, -1)                          # a row given once for all
    lens = torch.tensor([33 + t for t in range(tokens)], dtype=torch.int32, device="cuda")
    assert torch.equal(pkg.cache_attention(q[:tokens], cache, one, lens),
                       pkg.cache_attention(q[:tokens], cache, rows[:tokens].contiguous(), lens))
