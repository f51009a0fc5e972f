"""The MXFP8 cache on the GPU: rows written equal the quantizer's bytes, rows
read back equal the widened bytes, attention equals softmax(q K) V in 64 bits.
"""

import ctypes
import math

import numpy as np
import pytest
import torch

import MXFP8_quantizer

pytestmark = pytest.mark.gpu

pkg = MXFP8_quantizer.load_package()
capi = pkg._capi
TORCH = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
INDEX_BIT = 64


def raw(t):
    return t.view(torch.uint8)


def filled(pages, page, heads, dim, byte=0x7F, scale=255):
    """A cache whose every position decodes to NaN."""
    cache = pkg.allocate_cache(pages, page, heads, dim)
    raw(cache.k).fill_(byte), raw(cache.v).fill_(byte)
    cache.k_scales.fill_(scale), cache.v_scales.fill_(scale)
    return cache


def quantized(x):
    """(rows, heads, dim) -> payload bytes and scale bytes, by the library's own quantizer."""
    n, h, d = x.shape
    q, s = pkg.quantize(x.reshape(n * h, d), q_rows=n * h, q_cols=d)
    return raw(q).view(n, h, d), pkg.decode_scale_bytes(s, n * h, d).view(n, h, d // 32)


def widened(payload, scale):
    """float64 values of payload bytes (..., d) and scale bytes (..., d / 32)."""
    s = torch.exp2(scale.double() - 127)
    s[scale == 255] = math.nan
    return payload.view(torch.float8_e4m3fn).double() * s.repeat_interleave(32, -1)


def values(h, dim, n, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((n, h, dim), device="cuda", generator=g) * torch.exp2(3 * torch.randn((1, h, dim), device="cuda",
                                                                                          generator=g))
    return x.to(TORCH[dtype])


# --------------------------------------------------------------------------
# writing
# --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tokens,heads,dim,page", [(1, 1, 32, 1), (1, 8, 128, 16), (3, 3, 96, 4), (64, 8, 128, 16),
                                                   (65, 2, 256, 64), (200, 5, 64, 8), (513, 1, 160, 32),
                                                   (7, 2, 1024, 16)])
def test_write(tokens, heads, dim, page, dtype):
    pages = -(-tokens // page) + 3
    cache = filled(pages, page, heads, dim)
    k, v = values(heads, dim, tokens, dtype, 1), values(heads, dim, tokens, dtype, 2)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:tokens]
    slots[::7] = -1 - slots[::7]                                 # every seventh token is skipped
    want = [t.clone() for t in (raw(cache.k), raw(cache.v), cache.k_scales, cache.v_scales)]
    keep = slots >= 0
    at, off = slots[keep] // page, slots[keep] % page
    for x, w, ws in ((k, want[0], want[2]), (v, want[1], want[3])):
        if keep.any():
            w[at, :, off], ws[at, :, off] = quantized(x[keep])
    pkg.cache_write(cache, k, v, slots)
    for got, w in zip((raw(cache.k), raw(cache.v), cache.k_scales, cache.v_scales), want):
        assert torch.equal(got, w)
    assert capi.device_status() == 0


@pytest.mark.parametrize("offset", [0, 1, 8])
def test_write_reads_strided_rows_in_place(offset):
    """K and V as slices of one projection row, at any alignment; a transposed layout; one row for all tokens."""
    tokens, heads, dim = 33, 4, 64
    both = torch.randn((tokens, 2 * heads * dim + offset), device="cuda").bfloat16()
    k = both[:, offset:offset + heads * dim].view(tokens, heads, dim)
    v = both[:, offset + heads * dim:].view(tokens, heads, dim)
    slots = torch.arange(tokens, device="cuda")
    a, b, c, d = (filled(5, 8, heads, dim) for _ in range(4))
    pkg.cache_write(a, k, v, slots)
    pkg.cache_write(b, k.contiguous(), v.contiguous(), slots)
    pkg.cache_write(c, k.permute(1, 0, 2).contiguous().permute(1, 0, 2), v, slots)
    pkg.cache_write(d, k.permute(0, 2, 1).contiguous().permute(0, 2, 1), v, slots)   # copied: last dim strided
    for x, y, z, w in zip(a, b, c, d):
        assert torch.equal(raw(x), raw(y)) and torch.equal(raw(x), raw(z)) and torch.equal(raw(x), raw(w))
    one = k[:1].expand(tokens, heads, dim)
    pkg.cache_write(a, one, one, slots)
    payload, scale = quantized(k[:1])
    assert (raw(a.k)[0, :, 3] == payload[0]).all() and (a.v_scales[3, :, 7] == scale[0]).all()


def test_write_special_values():
    """Zero blocks, infs and NaNs get the quantizer's bytes."""
    x = torch.zeros((6, 1, 64), device="cuda", dtype=torch.bfloat16)
    x[1, 0, 3], x[2, 0, 40], x[3, 0, 0], x[4, 0, 33] = math.inf, math.nan, -math.inf, 3e38
    x[5] = 1e-38
    cache = filled(1, 8, 1, 64)
    pkg.cache_write(cache, x, x, torch.arange(6, device="cuda"))
    payload, scale = quantized(x)
    assert torch.equal(raw(cache.k)[0, 0, :6], payload[:, 0]) and torch.equal(cache.v_scales[0, 0, :6], scale[:, 0])


def test_write_skips_and_reports_slots_past_the_cache():
    cache = filled(3, 4, 2, 64)
    before = [raw(t).clone() for t in cache]
    x = torch.randn((4, 2, 64), device="cuda").half()
    pkg.cache_write(cache, x, x, torch.tensor([12, 2 ** 40, -(2 ** 40), 5], device="cuda"))
    assert capi.device_status(clear=True) == INDEX_BIT
    payload, scale = quantized(x)
    before[0][1, :, 1], before[2][1, :, 1] = payload[3], scale[3]
    before[1][1, :, 1], before[3][1, :, 1] = payload[3], scale[3]
    for t, w in zip(cache, before):
        assert torch.equal(raw(t), w)


# --------------------------------------------------------------------------
# reading back
# --------------------------------------------------------------------------

def random_cache(pages, page, heads, dim, seed, spread=4):
    """Finite random payloads, scale bytes 127 +- spread."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = pkg.allocate_cache(pages, page, heads, dim)
    for t in (cache.k, cache.v):
        b = torch.randint(0, 256, t.shape, device="cuda", generator=g, dtype=torch.int32).to(torch.uint8)
        raw(t).copy_(torch.where((b & 0x7F) == 0x7F, b - 1, b))
    for t in (cache.k_scales, cache.v_scales):
        t.copy_(torch.randint(127 - spread, 128 + spread, t.shape, device="cuda", generator=g, dtype=torch.int32))
    return cache


def random_table(lengths, page, pages, seed):
    """Distinct random pages; entries past a sequence's end are garbage."""
    g = torch.Generator().manual_seed(seed)
    width = max(1, max(-(-n // page) for n in lengths)) + 1
    table = torch.randint(-2 ** 31, 2 ** 31 - 1, (len(lengths), width), generator=g, dtype=torch.int64)
    order, at = torch.randperm(pages, generator=g), 0
    for b, n in enumerate(lengths):
        used = -(-n // page)
        table[b, :used] = order[at:at + used]
        at += used
    assert at <= pages
    return table.to(torch.int32).cuda()


def rows_of(payload, scale, table, b, n, page):
    """Sequence b's rows in 64 bits, (n, heads, dim)."""
    at = torch.arange(n, device="cuda")
    pages = table[b].long()[at // page]
    return widened(raw(payload)[pages, :, at % page], scale[pages, :, at % page])


@pytest.mark.parametrize("out", ["bf16", "fp16", "f32"])
@pytest.mark.parametrize("lengths,page,heads,dim", [([1], 1, 1, 32), ([5, 0, 17, 1], 4, 3, 96), ([0, 0], 16, 2, 64),
                                                    ([100, 33, 64, 7, 128], 16, 8, 128), ([300], 64, 2, 256)])
def test_read(lengths, page, heads, dim, out):
    pages = sum(-(-n // page) for n in lengths) + 2
    cache = random_cache(pages, page, heads, dim, dim)
    table = random_table(lengths, page, pages, 3)
    starts = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device="cuda")
    total = sum(lengths)
    k, v = pkg.cache_read(cache, table, starts, total, TORCH[out])
    for got, payload, scale in ((k, cache.k, cache.k_scales), (v, cache.v, cache.v_scales)):
        want = torch.cat([rows_of(payload, scale, table, b, n, page) for b, n in enumerate(lengths)])
        assert torch.equal(got, want.to(torch.float32).to(TORCH[out]))      # exact in f32, rounded once
    assert capi.device_status() == 0


def test_read_leaves_rows_that_no_sequence_covers():
    cache = random_cache(6, 4, 2, 64, 0)
    table = random_table([5, 3], 4, 6, 1)
    out = tuple(torch.full((14, 2, 64), -7.0, device="cuda") for _ in range(2))
    starts = torch.tensor([2, 7, 10], dtype=torch.int32, device="cuda")
    got = pkg.cache_read(cache, table, starts, 14, out=out)
    assert got[0] is out[0] and got[1] is out[1]
    want = torch.cat([rows_of(cache.k, cache.k_scales, table, b, n, 4) for b, n in ((0, 5), (1, 3))])
    assert torch.equal(out[0][2:10].double(), want)
    for t in out:
        assert (t[:2] == -7).all() and (t[10:] == -7).all()
    # a total below the sequences' end bounds the writes
    small = tuple(torch.full((9, 2, 64), -7.0, device="cuda") for _ in range(2))
    pkg.cache_read(cache, table, starts, 8, out=tuple(t[:8] for t in small))
    assert (small[0][8] == -7).all() and torch.equal(small[0][2:8], out[0][2:8])


def test_read_bad_pages_are_zeros_and_reported():
    cache = random_cache(6, 4, 2, 64, 0)
    table = torch.tensor([[0, -1, 6], [2 ** 31 - 1, 1, 2]], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 14, 26], dtype=torch.int32, device="cuda")    # sequence 0 runs past its table
    k, v = pkg.cache_read(cache, table, starts, 26, torch.float32)
    assert capi.device_status(clear=True) == INDEX_BIT
    for t in (k, v):
        assert (t[4:18] == 0).all()
    at = torch.arange(4, device="cuda")
    assert torch.equal(k[:4].double(), widened(raw(cache.k)[0][:, at], cache.k_scales[0][:, at]).transpose(0, 1))
    assert torch.equal(v[18:22].double(), widened(raw(cache.v)[1][:, at], cache.v_scales[1][:, at]).transpose(0, 1))


def test_read_shared_and_repeated_pages():
    """Two sequences over one prefix page, and a table row given once for all (stride 0)."""
    cache = random_cache(5, 8, 1, 64, 4)
    table = torch.tensor([[3, 1], [3, 3]], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 12, 28], dtype=torch.int32, device="cuda")
    k, _ = pkg.cache_read(cache, table, starts, 28)
    assert torch.equal(k[:8], k[12:20]) and torch.equal(k[12:20], k[20:28])
    same, _ = pkg.cache_read(cache, table[:1].expand(2, 2), torch.tensor([0, 12, 24], dtype=torch.int32, device="cuda"), 24)
    assert torch.equal(same[:12], k[:12]) and torch.equal(same[12:], k[:12])


# --------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------

def score_room(dim, size):
    """How far a score may be off, `size` being the largest scale * sum |q||k| of its head (see check_attention)."""
    return (dim + 32) * 2.0 ** -23 * size


def weight_room(err, n):
    """How far a weight times its V scale may be off, relative to it (see check_attention)."""
    return (2.0 ** -11 + 2 * (2 * err + 2.0 ** -20 + n * 2.0 ** -24)) * 1.01


def check_attention(q, cache, table, lengths, page, scale=None):
    """Against softmax in 64 bits.  Per head, with S the largest scale * sum |q||k|:
    scores are off by at most E = (dim + 32) 2^-23 S (an f32 sum of dim exact
    products, then a few f32 operations, each one unit in the last place of a
    partial sum), so a weight is off by a factor 2E + 2^-20 (exp2 and its
    argument's rounding, |argument| <= 2 S log2 e counted in E); the weight
    times the V scale is an f16, half a step 2^-11; sums of n terms add n 2^-24
    at most; f16 values below 2^-14 keep 2^-25 of the operand's unit, which is
    2^-15 of the largest V scale.  Then the output's rounding."""
    out, lse = pkg.cache_attention(q, cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), scale,
                                   return_lse=True)
    batch, q_heads, dim = q.shape
    heads = cache.k.shape[1]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    half = HALF_STEP[q.dtype]
    for b, n in enumerate(lengths):
        if n == 0:
            assert (out[b] == 0).all() and (lse[b] == -math.inf).all(), b
            continue
        k = rows_of(cache.k, cache.k_scales, table, b, n, page).repeat_interleave(q_heads // heads, 1)
        v = rows_of(cache.v, cache.v_scales, table, b, n, page).repeat_interleave(q_heads // heads, 1)
        s = scale * torch.einsum("hd,nhd->hn", q[b].double(), k)
        size = abs(scale) * torch.einsum("hd,nhd->hn", q[b].double().abs(), k.abs()).amax(1)
        err = score_room(dim, size)
        want_lse = torch.logsumexp(s, 1)
        p = torch.exp(s - want_lse[:, None])
        want = torch.einsum("hn,nhd->hd", p, v)
        weight = torch.einsum("hn,nhd->hd", p, v.abs())
        top = torch.exp2(cache.v_scales[table[b, :-(-n // page)].long()].double().amax() - 127)
        room = weight * weight_room(err, n)[:, None] + n * 448 * 2.0 ** -40 * top
        off = (out[b].double() - want).abs() - (room + half * (want.abs() + room) + 2.0 ** -25)
        assert not (off > 0).any(), (b, n, off.max().item(), weight.max().item())
        lse_off = (lse[b].double() - want_lse).abs() - (err + 2.0 ** -20 + n * 2.0 ** -24 + want_lse.abs() * 2.0 ** -22)
        assert not (lse_off > 0).any(), (b, n, lse_off.max().item())
    return out, lse


def attention_case(lengths, page, heads, group, dim, dtype, seed=0, spread=2):
    pages = sum(-(-n // page) for n in lengths) + 2
    cache = random_cache(pages, page, heads, dim, seed, spread)
    # payloads of +-448 at random scales give scores in the thousands: bring K to scores of a few
    cache.k_scales.sub_(8)
    table = random_table(lengths, page, pages, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = torch.randn((len(lengths), heads * group, dim), device="cuda", generator=g).to(TORCH[dtype])
    return q, cache, table


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 300, 1000]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,group,dim,page", [(1, 1, 64, 2), (2, 4, 64, 16), (3, 8, 128, 16), (1, 16, 128, 64),
                                                  (2, 5, 192, 8), (1, 7, 256, 32), (2, 12, 64, 8), (1, 24, 128, 16),
                                                  (1, 17, 256, 128), (8, 1, 128, 16)])
def test_attention(heads, group, dim, page, dtype):
    q, cache, table = attention_case(LENGTHS, page, heads, group, dim, dtype, seed=group + dim)
    check_attention(q, cache, table, LENGTHS, page)
    assert capi.device_status() == 0


@pytest.mark.parametrize("lengths,heads,group,dim", [([20000], 2, 4, 128), ([5000, 1, 0, 9001], 1, 8, 256),
                                                     ([64] * 300, 2, 2, 64), ([0] * 5, 2, 4, 128),
                                                     ([1] * 700, 1, 4, 64), ([3000] * 40, 4, 8, 128),
                                                     ([30000] + [3] * 300, 1, 4, 64), ([40000], 1, 1, 64)])
def test_attention_splits(lengths, heads, group, dim):
    """Few long sequences, many short ones, nothing at all."""
    q, cache, table = attention_case(lengths, 16, heads, group, dim, "bf16", seed=len(lengths))
    check_attention(q, cache, table, lengths, 16)
    assert capi.device_status() == 0


@pytest.mark.parametrize("batch", [31, 32, 33, 127, 128, 129])
def test_attention_batches(batch):
    """Around the batches at which a lane gets another sequence, and the join looks up where the pieces are."""
    lengths = [(37 * i) % 1500 if i % 5 else 0 for i in range(batch)]
    q, cache, table = attention_case(lengths, 16, 2, 4, 64, "bf16", seed=batch)
    check_attention(q, cache, table, lengths, 16)
    assert capi.device_status() == 0


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3])
def test_attention_scales(scale):
    q, cache, table = attention_case([100, 7], 8, 2, 4, 64, "bf16")
    check_attention(q, cache, table, [100, 7], 8, scale)


def test_attention_strided_queries():
    q, cache, table = attention_case([40, 70, 5], 16, 2, 4, 128, "bf16")
    want = pkg.cache_attention(q, cache, table, torch.tensor([40, 70, 5], dtype=torch.int32, device="cuda"))
    lengths = torch.tensor([40, 70, 5], dtype=torch.int32, device="cuda")
    wide = torch.zeros((3, 8, 131), device="cuda", dtype=torch.bfloat16)
    wide[:, :, 3:] = q
    for view in (wide[:, :, 3:], q.transpose(0, 1).contiguous().transpose(0, 1),
                 q.transpose(1, 2).contiguous().transpose(1, 2)):
        assert torch.equal(pkg.cache_attention(view, cache, table, lengths), want)


def test_attention_never_reads_what_is_not_there():
    """Positions past the end, other pages and table entries past the end hold NaN or garbage."""
    page, lengths = 16, [1, 33, 250, 0]
    pages = sum(-(-n // page) for n in lengths) + 2
    clean = random_cache(pages, page, 2, 128, 7)
    clean.k_scales.sub_(8)
    table = random_table(lengths, page, pages, 7)
    dirty = filled(pages, page, 2, 128)
    for b, n in enumerate(lengths):
        at = torch.arange(n, device="cuda")
        rows = table[b].long()[at // page]
        for d, c in zip(dirty, clean):
            raw(d)[rows, :, at % page] = raw(c)[rows, :, at % page]
    q = torch.randn((4, 8, 128), device="cuda").bfloat16()
    a, lse_a = check_attention(q, dirty, table, lengths, page)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    b, lse_b = pkg.cache_attention(q, clean, table, lens, return_lse=True)
    assert torch.equal(a, b) and torch.equal(lse_a, lse_b)
    assert capi.device_status() == 0


def test_attention_nan_reaches_what_it_belongs_to():
    q, cache, table = attention_case([200, 200], 16, 1, 4, 128, "bf16")
    lens = torch.tensor([200, 200], dtype=torch.int32, device="cuda")
    at = (int(table[0, 5]), 0, 3)                           # position 83 of sequence 0
    cache.v_scales[at][2] = 255                             # columns 64..95
    out = pkg.cache_attention(q, cache, table, lens)
    want = torch.zeros_like(out, dtype=torch.bool)
    want[0, :, 64:96] = True
    assert torch.equal(out.isnan(), want)
    raw(cache.v)[at][1] = 0x7F                              # and column 1
    want[0, :, 1] = True
    assert torch.equal(pkg.cache_attention(q, cache, table, lens).isnan(), want)
    cache.k_scales[at][0] = 255
    out, lse = pkg.cache_attention(q, cache, table, lens, return_lse=True)
    assert out[0].isnan().all() and lse[0].isnan().all() and not out[1].isnan().any()
    q[1, 2, 5] = math.nan
    out = pkg.cache_attention(q, cache, table, lens)
    assert out[1, 2].isnan().all() and not out[1, [0, 1, 3]].isnan().any()


def test_attention_wide_ranges():
    """V scales 2^24 apart between columns and positions, one dominant position, tiny and large queries."""
    lengths = [150, 150, 150]
    q, cache, table = attention_case(lengths, 16, 1, 4, 64, "bf16")
    g = torch.Generator(device="cuda").manual_seed(5)
    cache.v_scales.copy_(torch.randint(115, 140, cache.v_scales.shape, device="cuda", generator=g, dtype=torch.int32))
    q[0] *= 1e-30
    q[1] *= 8
    q[2, :, 1:] *= 2.0 ** -30
    check_attention(q, cache, table, lengths, 16)
    cache.v_scales.fill_(0)                                 # 2^-127
    out = pkg.cache_attention(q, cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    assert (out.abs() <= 448 * 2.0 ** -127).all()


def test_attention_a_scale_of_zero_before_a_large_one():
    """A first tile with scale bytes 0 does not disturb what follows."""
    lengths = [512]
    q, cache, table = attention_case(lengths, 16, 1, 2, 64, "bf16")
    for i in range(16):
        cache.v_scales[table[0, i].long()] = 0
    check_attention(q, cache, table, lengths, 16)


def test_attention_bad_pages_take_no_part():
    q, cache, table = attention_case([64, 100], 16, 2, 4, 64, "fp16")
    cut = table.clone()
    cut[1, 2] = 10 ** 6
    cut[1, 4] = -3
    lens = torch.tensor([64, 100], dtype=torch.int32, device="cuda")
    out, lse = pkg.cache_attention(q, cache, cut, lens, return_lse=True)
    assert capi.device_status(clear=True) == INDEX_BIT
    kept = torch.tensor([[0, 1, 3, 5, 6, 0]], dtype=torch.int32)
    short = table[1:, [0, 1, 3, 5, 6]].contiguous()         # 16 * 3 + 16 + 4 positions
    got, got_lse = pkg.cache_attention(q[1:], cache, short, torch.tensor([68], dtype=torch.int32, device="cuda"),
                                       return_lse=True)
    assert (lse[1] - got_lse[0]).abs().max() <= 2.0 ** -18 * (1 + got_lse.abs().max())
    assert (out[1].double() - got[0].double()).abs().max() <= 2.0 ** -9 * got.double().abs().max()
    gone = torch.full_like(table, -1)
    out, lse = pkg.cache_attention(q, cache, gone, lens, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    assert capi.device_status(clear=True) == INDEX_BIT
    # a length past the table is cut to it, a negative one is 0
    out, lse = pkg.cache_attention(q, cache, table[:, :3], torch.tensor([2 ** 31 - 1, -4], dtype=torch.int32,
                                                                       device="cuda"), return_lse=True)
    assert capi.device_status(clear=True) == INDEX_BIT
    want = pkg.cache_attention(q, cache, table[:, :3], torch.tensor([48, 0], dtype=torch.int32, device="cuda"))
    assert torch.equal(out, want) and (out[1] == 0).all()


def test_attention_without_pages():
    """An empty table and an empty cache: nothing to attend to, and a positive length is reported."""
    q = torch.randn((3, 4, 64), device="cuda").half()
    none = torch.empty((3, 0), dtype=torch.int32, device="cuda")
    zero, some = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.tensor([0, 5, 0], dtype=torch.int32, device="cuda")
    for cache in (pkg.allocate_cache(0, 16, 2, 64), filled(2, 16, 2, 64)):
        for lens, expect in ((zero, 0), (some, INDEX_BIT)):
            out, lse = pkg.cache_attention(q, cache, none, lens, return_lse=True)
            assert (out == 0).all() and (lse == -math.inf).all()
            assert capi.device_status(clear=True) == expect
    table = torch.zeros((3, 1), dtype=torch.int32, device="cuda")
    out = pkg.cache_attention(q, pkg.allocate_cache(0, 16, 2, 64), table, some)
    assert (out == 0).all() and capi.device_status(clear=True) == INDEX_BIT


def test_attention_lse_joins_two_halves():
    """A context attended to in two parts and joined by their lse equals the whole."""
    q, cache, table = attention_case([160], 16, 2, 4, 128, "bf16")
    def part(t, n):
        o, l = pkg.cache_attention(q, cache, t, torch.tensor([n], dtype=torch.int32, device="cuda"), return_lse=True)
        return o.double(), l.double()
    (o1, l1), (o2, l2), (o, l) = part(table[:, :6].contiguous(), 96), part(table[:, 6:10].contiguous(), 64), part(table, 160)
    w = torch.softmax(torch.stack([l1, l2]), 0)[..., None]
    assert (torch.logaddexp(l1, l2) - l).abs().max() <= 1e-5 * (1 + l.abs().max())
    top = torch.maximum(o1.abs(), o2.abs()).amax()
    assert (w[0] * o1 + w[1] * o2 - o).abs().max() <= 2 * 2.0 ** -8 * top


def test_streams_graphs_and_repeats():
    lengths = [900, 3, 0, 77]
    sets = [attention_case(lengths, 16, 2, 4, 128, "bf16", seed=s) for s in (1, 2)]
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 900, 903, 903, 980], dtype=torch.int32, device="cuda")
    want = [pkg.cache_attention(*s, lens, return_lse=True) for s in sets]
    want_rows = [pkg.cache_read(s[1], s[2], starts, 980) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    there = [pkg.cache_attention(*s, lens, return_lse=True, stream=side) for s in sets for _ in range(3)]
    rows = [pkg.cache_read(s[1], s[2], starts, 980, stream=side.cuda_stream) for s in sets]
    default = pkg.cache_attention(*sets[0], lens, stream=torch.cuda.default_stream())
    assert torch.equal(default, want[0][0])
    here = [pkg.cache_attention(*s, lens, return_lse=True) for s in sets for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    for i in range(6):
        for w, a, b in zip(want[i // 3], there[i], here[i]):
            assert torch.equal(w, a) and torch.equal(w, b)
    for w, r in zip(want_rows, rows):
        assert torch.equal(w[0], r[0]) and torch.equal(w[1], r[1])
    # a decode step captured once: write the new token, attend; replayed with new contents and lengths
    q, cache, table = sets[0]
    q, cache = q.clone(), pkg.MXFP8Cache(*(t.clone() for t in cache))
    new = torch.randn((4, 2, 128), device="cuda").bfloat16()
    slots = torch.full((4,), -1, device="cuda")
    steps = lens.clone()
    graph = torch.cuda.CUDAGraph()
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.cache_write(cache, new, new, slots)
        got = pkg.cache_attention(q, cache, table, steps, return_lse=True)
    with torch.cuda.graph(second):
        other = pkg.cache_attention(*sets[1], lens, return_lse=True)
    for step in range(3):
        new.normal_()
        slots.copy_(torch.stack([table[0, 56 + step // 16].long() * 16 + 4 + step, table[1, 0].long() * 16 + 3 + step,
                                 torch.tensor(-1, device="cuda"), table[3, 4].long() * 16 + 13 + step]))
        steps.copy_(torch.tensor([901 + step, 4 + step, 0, 78 + step]))
        graph.replay()
        second.replay()
        check = [t.clone() for t in got]
        fresh = pkg.MXFP8Cache(*(t.clone() for t in cache))
        pkg.cache_write(fresh, new, new, slots)
        for a, b in zip(check, pkg.cache_attention(q, fresh, table, steps, return_lse=True)):
            assert torch.equal(a, b)
        for a, b in zip(other, want[1]):
            assert torch.equal(a, b)
    assert capi.device_status() == 0


def test_a_decode_step_of_a_layer():
    """Projection in 4 bits, cache write, attention over what was written and read back: the operators in a row."""
    batch, heads, group, dim, page = 3, 2, 4, 64, 16
    width = 512
    x = torch.randn((batch, width), device="cuda").bfloat16()
    w = torch.randn(((heads * group + 2 * heads) * dim, width), device="cuda").bfloat16() / 16
    wq, ws = pkg.quantize_mxfp4(w)
    cache = filled(8, page, heads, dim)
    table = torch.tensor([[4, 1], [2, 0], [7, 3]], dtype=torch.int32, device="cuda")
    for step in range(20):
        xq, xs = pkg.quantize_mxfp4(x + step)
        y = pkg.mxfp4_gemm(xq, wq, xs, ws, torch.bfloat16)
        q, k, v = y.split([heads * group * dim, heads * dim, heads * dim], 1)
        slots = table[:, step // page].long() * page + step % page
        pkg.cache_write(cache, k.view(batch, heads, dim), v.view(batch, heads, dim), slots)
        lengths = torch.full((batch,), step + 1, dtype=torch.int32, device="cuda")
        out = pkg.cache_attention(q.view(batch, heads * group, dim), cache, table, lengths)
    starts = torch.arange(batch + 1, dtype=torch.int32, device="cuda") * 20
    rows_k, rows_v = (t.view(batch, 20, heads, dim).double() for t in pkg.cache_read(cache, table, starts, 60, torch.float32))
    rk, rv = (t.repeat_interleave(group, 2) for t in (rows_k, rows_v))
    s = torch.einsum("bhd,bnhd->bhn", q.view(batch, heads * group, dim).double(), rk) / math.sqrt(dim)
    p = torch.softmax(s, -1)
    want, weight = torch.einsum("bhn,bnhd->bhd", p, rv), torch.einsum("bhn,bnhd->bhd", p, rv.abs())
    # the scores are in the thousands, so their rounding is not small: score_room's bound, which for
    # scores of 6000 is 0.07, and the output's half step
    size = torch.einsum("bhd,bnhd->bhn", q.view(batch, heads * group, dim).double().abs(), rk.abs()) / math.sqrt(dim)
    top = torch.exp2(cache.v_scales[table.long()].double().amax() - 127)
    room = weight * weight_room(score_room(dim, size.amax(-1)), 20)[..., None] + 20 * 448 * 2.0 ** -40 * top
    off = (out.double() - want).abs() - (room + 2.0 ** -8 * (want.abs() + room))
    worst = off.argmax()
    assert not (off > 0).any(), [t.flatten()[worst].item() for t in (off, out, want, weight)]
    assert capi.device_status() == 0


@pytest.mark.slow
def test_a_cache_past_32_bit_offsets():
    """Pages whose byte offsets pass 2^32."""
    pages, page, heads, dim = 2 ** 22 + 40, 16, 1, 64       # 4.3 GB of K, as much of V
    cache = pkg.MXFP8Cache(torch.empty((pages, heads, page, dim), dtype=torch.float8_e4m3fn, device="cuda"),
                           torch.empty((pages, heads, page, dim), dtype=torch.float8_e4m3fn, device="cuda"),
                           torch.empty((pages, heads, page, dim // 32), dtype=torch.uint8, device="cuda"),
                           torch.empty((pages, heads, page, dim // 32), dtype=torch.uint8, device="cuda"))
    table = torch.tensor([[pages - 1, 3, 2 ** 22 + 1, 2 ** 21]], dtype=torch.int32, device="cuda")
    small = filled(4, page, heads, dim)
    near = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    k, v = (torch.randn((64, heads, dim), device="cuda").bfloat16() for _ in range(2))
    at = torch.arange(64, device="cuda")
    pkg.cache_write(cache, k, v, table[0].long()[at // page] * page + at % page)
    pkg.cache_write(small, k, v, at)
    starts = torch.tensor([0, 64], dtype=torch.int32, device="cuda")
    for a, b in zip(pkg.cache_read(cache, table, starts, 64), pkg.cache_read(small, near, starts, 64)):
        assert torch.equal(a, b)
    q = torch.randn((1, 4, dim), device="cuda").bfloat16()
    lens = torch.tensor([64], dtype=torch.int32, device="cuda")
    assert torch.equal(pkg.cache_attention(q, cache, table, lens), pkg.cache_attention(q, small, near, lens))
    assert capi.device_status() == 0


def test_checked_build():
    """Every store of the checked build lies in its output; narrowed windows show that the guards see these kernels."""
    checked = capi.checked_lib()
    word = ctypes.c_uint32(0)
    stream = torch.cuda.current_stream().cuda_stream
    lengths, page, heads, dim = [70, 0, 16 * 30], 16, 2, 128
    q, cache, table = attention_case(lengths, page, heads, 4, dim, "bf16")
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 70, 70, 550], dtype=torch.int32, device="cuda")
    pages = cache.k.shape[0]
    copy = pkg.MXFP8Cache(*(t.clone() for t in cache))
    x = torch.randn((pages * page, heads, dim), device="cuda").bfloat16()
    slots = torch.arange(pages * page, device="cuda")
    pkg.cache_write(cache, x, x, slots)
    want = pkg.cache_attention(q, cache, table, lens)
    rows = pkg.cache_read(cache, table, starts, 550)
    d = capi.Cache(*(t.data_ptr() for t in copy), pages, heads, page, dim)
    out, k_out, v_out = torch.zeros_like(want), torch.zeros_like(rows[0]), torch.zeros_like(rows[1])
    size = capi.cache_attention_workspace(d, 3, 8)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")

    def call_all():
        yield checked.mxfp8_cache_write(d, x.data_ptr(), 256, 128, x.data_ptr(), 256, 128, 0, slots.numel(),
                                        slots.data_ptr(), stream)
        yield checked.mxfp8_cache_read(d, table.data_ptr(), table.stride(0), table.shape[1], 3, starts.data_ptr(), 550,
                                       k_out.data_ptr(), v_out.data_ptr(), 0, stream)
        yield checked.mxfp8_cache_attention(d, q.data_ptr(), q.stride(0), q.stride(1), 0, 3, 8, table.data_ptr(),
                                            table.stride(0), table.shape[1], lens.data_ptr(), dim ** -0.5,
                                            out.data_ptr(), None, ws.data_ptr(), size, stream)

    for slack, expect in ((0, 0), (64, 16)):
        assert checked.mxfp8_checked_window_slack(slack) == 0
        for rc in call_all():
            assert rc == 0
            assert checked.mxfp8_device_status(ctypes.byref(word), 1) == 0
            assert word.value == expect
    assert checked.mxfp8_checked_window_slack(0) == 0
    assert torch.equal(out, want) and torch.equal(k_out, rows[0]) and torch.equal(v_out, rows[1])
    for a, b in zip(copy, cache):
        assert torch.equal(raw(a), raw(b))
    assert checked.mxfp8_cache_attention(d, q.data_ptr(), q.stride(0), q.stride(1), 0, 3, 8, table.data_ptr(),
                                         table.stride(0), table.shape[1], lens.data_ptr(), 1.0, out.data_ptr(), None,
                                         ws.data_ptr(), size - 1, stream) == capi.ERR_WORKSPACE
