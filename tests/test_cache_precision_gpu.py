"""cache_attention's weights hold more bits than one f16: rows of V that nearly
cancel show them, as the output's own rounding is then small."""

import math

import pytest
import torch

from test_cache_gpu import HALF_STEP, TORCH, attention_case, capi, pkg, raw, rows_of, score_room

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,group,dim", [(4, 8, 64), (2, 16, 64), (4, 8, 128), (2, 16, 128), (4, 8, 192), (4, 8, 256)])
@pytest.mark.parametrize("n", [2, 3, 8, 40])
def test_weights_of_rows_that_cancel(n, heads, group, dim, dtype):
    """V rows +x and -x in turn.  Per element, relative to sum p |v|: scores are
    off by E = score_room, a weight by a factor 2 E + 2^-20 (exp2 and its
    argument), its two f16 by 2^-22, sums of n terms by n 2^-24, and as much
    again in the softmax's sum; then half a step of the output.  One f16 alone
    would be off by 2^-11."""
    lengths = [n] * 4
    q, cache, table = attention_case(lengths, 64, heads, group, dim, dtype, seed=n + dim, spread=0)
    raw(cache.v)[:, :, 0::2] = raw(cache.v)[:, :, 0:1] & 0x7F
    raw(cache.v)[:, :, 1::2] = raw(cache.v)[:, :, 0:1] | 0x80
    scale = 0.02 / math.sqrt(dim)                              # scores below 1: E stays below 2^-14
    out = pkg.cache_attention(q, cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), scale)
    for b in range(4):
        k = rows_of(cache.k, cache.k_scales, table, b, n, 64).repeat_interleave(group, 1)
        v = rows_of(cache.v, cache.v_scales, table, b, n, 64).repeat_interleave(group, 1)
        err = score_room(dim, scale * torch.einsum("hd,nhd->hn", q[b].double().abs(), k.abs()).amax(1))
        assert (err < 2.0 ** -14).all()
        p = torch.softmax(scale * torch.einsum("hd,nhd->hn", q[b].double(), k), 1)
        want = torch.einsum("hn,nhd->hd", p, v)
        rel = 2.0 ** -22 + 2 * (2 * err + 2.0 ** -20 + n * 2.0 ** -24)
        room = torch.einsum("hn,nhd->hd", p, v.abs()) * rel[:, None] * 1.01
        room = room + HALF_STEP[TORCH[dtype]] * (want.abs() + room) + 2.0 ** -25
        off = (out[b].double() - want).abs()
        assert out[b].isfinite().all() and (off <= room).all(), (b, (off / room).max().item())
    assert capi.device_status() == 0
