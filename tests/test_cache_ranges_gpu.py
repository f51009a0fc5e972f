"""cache_attention where V's scales lie far apart: between columns, between
positions, beside rows of zeros (whose blocks have scale byte 127), and at the
ends of their range.  Each output element is held to its own terms."""

import math

import pytest
import torch

import MXFP8_quantizer
from test_cache_gpu import (HALF_STEP, TORCH, attention_case, capi, filled, pkg, random_table, raw, rows_of, score_room,
                            weight_room)

pytestmark = pytest.mark.gpu

SMALLEST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}   # half the least value


def check_elements(q, cache, table, lengths, page, scale=None):
    """Against softmax in 64 bits.  A weight is off by weight_room relative to
    itself (test_cache_gpu.py), or where f16 has no more bits by half its least
    step, 2^-25, in units in which the largest weight beside the window's
    largest V scale is 2^15.  A window takes V scales 2^11 apart at most, so that
    is 2^-29 of the largest weight, times the element's own |v|.  Windows go
    down to 2^-64 of the largest V scale met; below, the step is 2^-104 of it."""
    out, lse = pkg.cache_attention(q, cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), scale,
                                   return_lse=True)
    dim, group = q.shape[2], q.shape[1] // cache.k.shape[1]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    half = HALF_STEP[q.dtype]
    for b, n in enumerate(lengths):
        k = rows_of(cache.k, cache.k_scales, table, b, n, page).repeat_interleave(group, 1)
        v = rows_of(cache.v, cache.v_scales, table, b, n, page).repeat_interleave(group, 1)
        s = scale * torch.einsum("hd,nhd->hn", q[b].double(), k)
        err = score_room(dim, abs(scale) * torch.einsum("hd,nhd->hn", q[b].double().abs(), k.abs()).amax(1))
        want_lse = torch.logsumexp(s, 1)
        p = torch.exp(s - want_lse[:, None])
        want = torch.einsum("hn,nhd->hd", p, v)
        top = torch.exp2(cache.v_scales[table[b, :-(-n // page)].long()].double().amax() - 127)
        room = (torch.einsum("hn,nhd->hd", p, v.abs()) * weight_room(err, n)[:, None]
                + p.amax(1)[:, None] * 2.0 ** -29 * v.abs().sum(0) + n * 448 * 2.0 ** -104 * top)
        room = room + half * (want.abs() + room) + SMALLEST[q.dtype]
        off = (out[b].double() - want).abs()
        assert out[b].isfinite().all() and lse[b].isfinite().all()
        assert (off <= room).all(), (b, n, (off / room).max().item(), want.abs().max().item())
        lse_room = err + 2.0 ** -20 + n * 2.0 ** -24 + want_lse.abs() * 2.0 ** -22
        assert ((lse[b].double() - want_lse).abs() <= lse_room).all(), (b, n)
    assert capi.device_status() == 0
    return out


@pytest.mark.parametrize("heads,group,dim", [(2, 4, 64), (1, 12, 64), (2, 3, 128), (1, 16, 128), (1, 4, 192), (1, 8, 256)])
@pytest.mark.parametrize("low", [126, 115, 98, 80, 64])
def test_column_blocks_far_apart(heads, group, dim, low):
    """One block of columns at scale byte 127, the others around `low`."""
    lengths = [1, 33, 700, 16]
    q, cache, table = attention_case(lengths, 16, heads, group, dim, "bf16", seed=low, spread=1)
    cache.v_scales.sub_(127 - low)
    cache.v_scales[..., 1] = 127
    check_elements(q, cache, table, lengths, 16)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("size", [1.0, 1e-5, 1e-6, 1e-7])
def test_zero_rows_among_small_ones(size, dtype):
    """Rows of zeros written beside rows of `size`; the position that takes nearly all of the weight is one of them."""
    lengths, page, heads, group, dim = [4096, 200], 16, 2, 4, 128
    g = torch.Generator(device="cuda").manual_seed(7)
    total = sum(lengths)
    k, v = (torch.randn((total, heads, dim), device="cuda", generator=g) for _ in range(2))
    v = v * size * (1 if dtype == "bf16" else 32)                       # fp16 has no fewer bits there
    v[::9] = 0
    q = torch.randn((2, heads * group, dim), device="cuda", generator=g)
    k[0], k[4096] = (q[b].view(heads, group, dim).sum(1) * (8 * math.sqrt(dim) / (q[b] * q[b]).sum(-1).mean()) for b in (0, 1))
    pages = -(-4096 // page) + -(-200 // page) + 2
    cache, table = filled(pages, page, heads, dim), random_table(lengths, page, pages, 1)
    slots = torch.cat([table[b].long()[torch.arange(n, device="cuda") // page] * page + torch.arange(n, device="cuda") % page
                       for b, n in enumerate(lengths)])
    pkg.cache_write(cache, k.to(TORCH[dtype]), v.to(TORCH[dtype]), slots)
    check_elements(q.to(TORCH[dtype]), cache, table, lengths, page)


@pytest.mark.parametrize("heads,group,dim", [(2, 4, 64), (1, 8, 128), (1, 16, 128), (1, 5, 192), (1, 8, 256)])
@pytest.mark.parametrize("low,high", [(100, 140), (80, 160), (121, 133), (1, 40), (60, 200)])
def test_positions_and_blocks_at_any_scale(low, high, heads, group, dim):
    """Every block a scale of its own: several windows a tile, pieces joined over warps and CTAs."""
    lengths = [6000, 31, 2, 400]
    q, cache, table = attention_case(lengths, 16, heads, group, dim, "bf16", seed=low)
    g = torch.Generator(device="cuda").manual_seed(low)
    cache.v_scales.copy_(torch.randint(low, high, cache.v_scales.shape, device="cuda", generator=g, dtype=torch.int32))
    check_elements(q, cache, table, lengths, 16)


def test_small_weights_beside_the_largest_scales():
    """V near the end of f32: the weights that count are 2^-20 and less, the one near 1 meets a row of zeros."""
    lengths, dim = [700], 64
    q, cache, table = attention_case(lengths, 16, 1, 2, dim, "bf16", seed=3)
    raw(cache.v).bitwise_and_(0x9F)                                     # |payload| below 2^-2
    cache.v_scales.fill_(250)
    k = rows_of(cache.k, cache.k_scales, table, 0, 700, 16)
    s = torch.einsum("hd,nhd->hn", q[0].double(), k) / math.sqrt(dim)
    best = s.amax(0).argmax().item()
    raw(cache.v)[table[0, best // 16].long(), :, best % 16] = 0
    scale = 20.0 / (s.amax(1) - s.median(1).values).amin().item() / math.sqrt(dim)
    out = check_elements(q, cache, table, lengths, 16, scale)
    assert (out != 0).all()


def test_nan_scales_beside_several_windows():
    """A NaN block reaches its columns alone, also where a tile's other scales take several windows."""
    lengths = [200, 64]
    q, cache, table = attention_case(lengths, 16, 1, 4, 128, "bf16")
    g = torch.Generator(device="cuda").manual_seed(0)
    cache.v_scales.copy_(torch.randint(60, 180, cache.v_scales.shape, device="cuda", generator=g, dtype=torch.int32))
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    clean = pkg.cache_attention(q, cache, table, lens)
    cache.v_scales[int(table[0, 5]), 0, 3, 2] = 255
    out = pkg.cache_attention(q, cache, table, lens)
    nan = torch.zeros_like(out, dtype=torch.bool)
    nan[0, :, 64:96] = True
    assert torch.equal(out.isnan(), nan)
    assert torch.equal(out[1], clean[1])
    cache.v_scales[table[1, :4].long()] = 255                            # nothing but NaN
    assert pkg.cache_attention(q, cache, table, lens)[1].isnan().all()


def test_windows_do_not_depend_on_what_is_absent():
    """A sequence's last tile holds positions past its end at other scales: the same bits as without them."""
    lengths = [5, 37]
    q, cache, table = attention_case(lengths, 16, 2, 4, 64, "bf16", seed=9)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = pkg.cache_attention(q, cache, table, lens, return_lse=True)
    for byte in (0, 90, 200, 255):
        cache.v_scales[table[0, 0].long(), :, 5:] = byte
        cache.v_scales[table[1, 2].long(), :, 5:] = byte
        for a, b in zip(pkg.cache_attention(q, cache, table, lens, return_lse=True), want):
            assert torch.equal(a, b)


def test_a_scale_without_a_payload_takes_nothing():
    """Zero payloads under the largest scale beside ordinary rows and very small ones, in one tile."""
    lengths = [32, 100]
    q, cache, table = attention_case(lengths, 16, 1, 4, 64, "bf16", seed=12)
    for low in (127, 60, 20, 5):
        cache.v_scales.fill_(low)
        at = table[:, 0].long()
        raw(cache.v)[at, :, 3:9] = 0
        cache.v_scales[at, :, 3:9] = 254
        check_elements(q, cache, table, lengths, 16)
