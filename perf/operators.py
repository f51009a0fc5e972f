"""The workloads of the 4-bit and cache operators: their cases, inputs, plain
forms and 64-bit values.

Five operators, in the order a served layer meets them:

- ``mxfp4``      quantize_mxfp4 then dequantize_mxfp4: E2M1 codes with one UE8M0
                 scale per 1x32 block, and the values they stand for.
- ``gemm``       mxfp4_gemm: C = A B^T of two MXFP4 matrices.
- ``write``      cache_write: K and V rows quantized into MXFP8 pages.
- ``read``       cache_read: the rows of a batch's pages, widened and packed.
- ``attention``  cache_attention: one query token per sequence over the pages.

With ``own`` false ``run`` computes the plain form (elementary torch operations
in 32 bits); with ``own`` true it calls the framework.
"""

import math

import torch

own = False

BLOCK = 32                     # elements that share one scale
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "f32": 4}


def listed():
    return [
        # a ragged batch of activations (the odd-sized layer of the repository's fp16 tests)
        dict(name="mxfp4 1000x4064 fp16", op="mxfp4", m=1000, k=4064, dtype="fp16", out="fp16"),
        # a weight matrix converted when a checkpoint is loaded
        dict(name="mxfp4 8192x8192 bf16", op="mxfp4", m=8192, k=8192, dtype="bf16", out="bf16"),
        # one decoded token through a 4-bit projection
        dict(name="gemm 1x4096x4096", op="gemm", m=1, n=4096, k=4096, out="bf16"),
        # a small ragged batch, odd output width, unrounded sums
        dict(name="gemm 77x1000x2080 f32", op="gemm", m=77, n=1000, k=2080, out="f32"),
        # prefill of 8192 tokens through a wide projection
        dict(name="gemm 8192x8192x8192", op="gemm", m=8192, n=8192, k=8192, out="bf16"),
        # the new token of each of 64 sequences
        dict(name="write 64 tokens", op="write", tokens=64, heads=8, dim=128, page=16, dtype="bf16", skip=False),
        # a packed prefill batch whose padding rows carry no slot
        dict(name="write 8191 tokens", op="write", tokens=8191, heads=8, dim=128, page=16, dtype="bf16", skip=True),
        # a short prefix read back before a chunk of prefill
        dict(name="read 5x257", op="read", batch=5, longest=257, heads=4, dim=64, page=8, out="fp16"),
        # the prefixes of a whole batch
        dict(name="read 32x4096", op="read", batch=32, longest=4096, heads=8, dim=128, page=16, out="bf16"),
        # one user's next token
        dict(name="attention 1x1000", op="attention", batch=1, longest=1000, groups=4, heads=8, dim=128, page=16,
             dtype="bf16", empty=False),
        # a ragged serving batch with idle rows
        dict(name="attention 64x4096 ragged", op="attention", batch=64, longest=4096, groups=4, heads=8, dim=128,
             page=16, dtype="bf16", empty=True),
        # long contexts, few wide heads
        dict(name="attention 8x65536", op="attention", batch=8, longest=65536, groups=8, heads=2, dim=256, page=64,
             dtype="fp16", empty=False),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["mxfp4", "gemm", "write", "read", "attention"])
    if op == "mxfp4":
        dtype = rng.choice(["bf16", "fp16"])
        k = _spread(rng, 1, 8192)
        return dict(op=op, m=_spread(rng, 1, 8192), k=k, dtype=dtype, out=rng.choice(["bf16", "fp16", "f32"]))
    if op == "gemm":
        return dict(op=op, m=_spread(rng, 1, 8192), n=_spread(rng, 1, 8192), k=BLOCK * _spread(rng, 1, 256),
                    out=rng.choice(["bf16", "fp16", "f32"]))
    if op == "write":
        return dict(op=op, tokens=_spread(rng, 1, 8192), heads=rng.choice([1, 2, 3, 4, 8]),
                    dim=rng.choice([32, 64, 96, 128]), page=rng.choice([1, 8, 16, 32, 64]),
                    dtype=rng.choice(["bf16", "fp16"]), skip=rng.random() < 0.5)
    longest = _spread(rng, 1, 32768)
    batch = min(_spread(rng, 1, 128), max(1, 131072 // longest))
    if op == "read":
        return dict(op=op, batch=batch, longest=longest, heads=rng.choice([1, 2, 3, 4]),
                    dim=rng.choice([32, 64, 96, 128]), page=rng.choice([1, 8, 16, 32, 64]),
                    out=rng.choice(["bf16", "fp16", "f32"]))
    heads, groups = rng.choice([(8, 1), (8, 4), (8, 8), (4, 5), (2, 7), (2, 16), (1, 16), (1, 24)])
    return dict(op=op, batch=batch, longest=longest, groups=groups, heads=heads,
                dim=rng.choice([64, 128, 192, 256] if heads < 8 else [64, 128]), page=rng.choice([8, 16, 32, 64, 128]),
                dtype=rng.choice(["bf16", "fp16"]), empty=rng.random() < 0.5)


# --------------------------------------------------------------------------
# the formats
# --------------------------------------------------------------------------

def _ceil(a, b):
    return -(-a // b) * b


def _mxfp4_parts(x):
    """(m, k) values, k a multiple of 32 -> signed E2M1 values f32 (m, k) and scale bytes (m, k/32)."""
    m, k = x.shape
    v = x.float().view(m, k // BLOCK, BLOCK)
    amax = v.abs().amax(-1)
    f, p = torch.frexp(amax)                              # amax = f 2^p; 6 2^e = 0.75 2^(e+3)
    e = (p - 3 + (f > 0.75).int()).clamp(min=-127)
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    y = v * torch.exp2(-e.float())[..., None]
    a = y.abs()
    # nearest of 0 .5 1 1.5 2 3 4 6; a value midway goes to the code whose last bit is 0
    mag = (0.5 * ((a > 0.25).float() + (a >= 0.75).float() + (a > 1.25).float() + (a >= 1.75).float())
           + (a > 2.5).float() + (a >= 3.5).float() + 2.0 * (a > 5.0).float())
    return torch.where(y < 0, -mag, mag).view(m, k), (e + 127).to(torch.uint8)


def _chunk_index(rows, blocks, device):
    """Byte offset of scale (row, block) in the 128-row x 4-block chunks of 512 bytes."""
    r = torch.arange(rows, device=device)[:, None]
    c = torch.arange(blocks, device=device)[None, :]
    chunk = (r // 128) * (-(-blocks // 4)) + c // 4
    return chunk * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + c % 4


def _pack_scales(dense):
    rows, blocks = dense.shape
    out = torch.zeros(_ceil(rows, 128) * _ceil(blocks, 4), dtype=torch.uint8, device=dense.device)
    out[_chunk_index(rows, blocks, dense.device).view(-1)] = dense.reshape(-1)
    return out


def _power(byte):
    """2^(byte - 127) of scale bytes, in 32 bits."""
    return torch.exp2(byte.float() - 127.0)


def _pack_codes(values):
    """Signed E2M1 values (m, k) -> bytes (m, k/2), the even element in the low half."""
    a = values.abs()
    code = torch.where(a <= 2, 2 * a, torch.where(a <= 4, a + 2, a + 1)).to(torch.uint8)
    code = code | ((values < 0).to(torch.uint8) << 3)
    return code[:, 0::2] | (code[:, 1::2] << 4)


def _codes_to_values(packed):
    """Bytes (m, k/2) -> E2M1 values (m, k)."""
    code = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    low = (code & 7).float()
    mag = torch.where(low <= 4, 0.5 * low, torch.where(low <= 6, low - 2, low - 1))
    return torch.where(code >= 8, -mag, mag)


def _mxfp8_parts(x):
    """(..., d) values, d a multiple of 32 -> E4M3 values and scale bytes (..., d/32)."""
    v = x.float().unflatten(-1, (-1, BLOCK))
    amax = v.abs().amax(-1)
    # amax/448 + 1e-12 with both constants in 32 bits, rounded once, then up to a power of two
    c = torch.tensor(1.0 / 448.0, dtype=torch.float32).item()
    eps = torch.tensor(1.0e-12, dtype=torch.float32).item()
    bits = (amax.double() * c + eps).float().view(torch.int32)
    byte = (bits >> 23) + ((bits & 0x7FFFFF) != 0).int()
    byte = torch.where(amax == 0, torch.full_like(byte, 127), byte)
    y = v * torch.exp2(127.0 - byte.float())[..., None]
    return y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).flatten(-2), byte.to(torch.uint8)


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def _lengths(case):
    """The batch's lengths: spread over 1..longest, the longest among them, every eighth one 0 where `empty`."""
    n, top = case["batch"], case["longest"]
    out = [max(1, int(round(top * ((b * 0.6180339887498949 + 1.0) % 1.0 or 1.0)))) for b in range(n)]
    out[0] = top
    if case.get("empty"):
        out = [0 if b % 8 == 5 or (n > 1 and b == n - 1 and n < 6) else v for b, v in enumerate(out)]
    return out


def _paged(case, gen):
    """Pages with quantized contents, and a table that scatters the batch's pages over them."""
    heads, dim, page = case["heads"], case["dim"], case["page"]
    lengths = _lengths(case)
    per = -(-case["longest"] // page)
    need = sum(-(-v // page) for v in lengths)
    pages = need + 3
    cache = []
    for _ in range(2):
        spread = torch.exp2(torch.randn((1, heads, 1, dim), device="cuda", generator=gen))
        x = torch.randn((pages, heads, page, dim), device="cuda", generator=gen, dtype=torch.float32)
        cache += list(_mxfp8_parts((x * spread).bfloat16()))
        del x
    order = torch.randperm(pages, device="cuda", generator=gen, dtype=torch.int32)
    table = torch.zeros((case["batch"], per), device="cuda", dtype=torch.int32)
    lens = torch.tensor(lengths, device="cuda", dtype=torch.int64)
    lens = lens[torch.randperm(case["batch"], device="cuda", generator=gen)]
    used = (lens + page - 1) // page
    mask = torch.arange(per, device="cuda")[None, :] < used[:, None]
    table[mask] = order[:need]
    return (cache[0], cache[2], cache[1], cache[3]), table, lens


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    state = dict(case=case)

    def normal(*shape, dtype):
        return torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32).to(dtype)

    if op == "mxfp4":
        # outlier channels, as activations and weights have them
        spread = torch.exp2(2.0 * torch.randn((1, case["k"]), device="cuda", generator=gen))
        x = torch.randn((case["m"], case["k"]), device="cuda", generator=gen)
        state["x"] = (x * spread).clamp(-3e4, 3e4).to(TYPES[case["dtype"]])
    elif op == "gemm":
        for name, rows in (("a", case["m"]), ("b", case["n"])):
            values, byte = _mxfp4_parts(normal(rows, case["k"], dtype=torch.bfloat16) * (1.0 if name == "a" else 0.02))
            state[name + "_q"] = _pack_codes(values)
            state[name + "_s"] = _pack_scales(byte)
    elif op == "write":
        tokens, heads, dim, page = case["tokens"], case["heads"], case["dim"], case["page"]
        dtype = TYPES[case["dtype"]]
        pages = -(-tokens // page) + 5
        # K and V as a fused projection leaves them: two slices of one row
        both = normal(tokens, 2 * heads * dim, dtype=dtype)
        state["k"] = both[:, :heads * dim].view(tokens, heads, dim)
        state["v"] = both[:, heads * dim:].view(tokens, heads, dim)
        state["slots"] = torch.randperm(pages * page, device="cuda", generator=gen)[:tokens]
        if case["skip"]:
            state["slots"][torch.rand(tokens, device="cuda", generator=gen) < 0.1] = -1
        old = [_mxfp8_parts(normal(pages, heads, page, dim, dtype=dtype)) for _ in range(2)]
        state["cache"] = (old[0][0], old[1][0], old[0][1], old[1][1])
    elif op == "read":
        state["cache"], state["table"], lens = _paged(case, gen)
        state["starts"] = torch.cat((lens.new_zeros(1), lens.cumsum(0))).to(torch.int32)
        state["total"] = sum(_lengths(case))
    else:
        state["cache"], state["table"], lens = _paged(case, gen)
        state["lengths"] = lens.to(torch.int32)
        state["q"] = normal(case["batch"], case["heads"] * case["groups"], case["dim"], dtype=TYPES[case["dtype"]])
    return state


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def _gathered(pages, scales, table, length):
    """Rows 0..length-1 of every sequence, widened: (batch, length, heads, dim) f32."""
    page = pages.shape[2]
    at = torch.arange(length, device=table.device)
    which, offset = table[:, at // page].long(), at % page
    q = pages.view(torch.uint8)[which, :, offset].view(torch.float8_e4m3fn).float()
    s = _power(scales[which, :, offset])
    return (q.unflatten(-1, (-1, BLOCK)) * s[..., None]).flatten(-2)


def _plain(state):
    case = state["case"]
    op = case["op"]
    if op == "mxfp4":
        x = state["x"]
        x = torch.nn.functional.pad(x, (0, _ceil(case["k"], BLOCK) - case["k"]))
        values, byte = _mxfp4_parts(x)
        out = values.unflatten(-1, (-1, BLOCK)) * _power(byte)[..., None]
        return {"values": out.flatten(-2).to(TYPES[case["out"]]), "scales": _pack_scales(byte)}
    if op == "gemm":
        sides = []
        for name, rows in (("a", case["m"]), ("b", case["n"])):
            s = state[name + "_s"][_chunk_index(rows, case["k"] // BLOCK, "cuda")]
            v = _codes_to_values(state[name + "_q"]).unflatten(-1, (-1, BLOCK)) * _power(s)[..., None]
            sides.append(v.flatten(-2))
        return (sides[0] @ sides[1].t()).to(TYPES[case["out"]])
    if op == "write":
        slots, page = state["slots"], case["page"]
        keep = slots >= 0
        slots = slots[keep]
        for x, pages, scales in (("k", 0, 2), ("v", 1, 3)):
            q, byte = _mxfp8_parts(state[x][keep])
            state["cache"][pages].view(torch.uint8)[slots // page, :, slots % page] = q.view(torch.uint8)
            state["cache"][scales][slots // page, :, slots % page] = byte
        return state["cache"]
    if op == "read":
        k_pages, v_pages, k_scales, v_scales = state["cache"]
        starts, longest = state["starts"].long(), case["longest"]
        mask = torch.arange(longest, device="cuda")[None, :] < (starts[1:] - starts[:-1])[:, None]
        return tuple(_gathered(p, s, state["table"], longest)[mask].to(TYPES[case["out"]])
                     for p, s in ((k_pages, k_scales), (v_pages, v_scales)))
    k_pages, v_pages, k_scales, v_scales = state["cache"]
    lens, longest = state["lengths"], case["longest"]
    q = state["q"].float().unflatten(1, (case["heads"], case["groups"]))
    k = _gathered(k_pages, k_scales, state["table"], longest)
    live = (torch.arange(longest, device="cuda")[None, :] < lens[:, None])[:, None, None, :]
    score = torch.matmul(q, k.permute(0, 2, 3, 1)) / math.sqrt(case["dim"])     # (batch, heads, groups, length)
    del k
    score = torch.where(live, score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    v = _gathered(v_pages, v_scales, state["table"], longest)
    out = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + torch.log(total)).flatten(1)
    return {"out": out.flatten(1, 2).to(TYPES[case["dtype"]]), "lse": lse}


_package = None


def _own(state):
    global _package
    if _package is None:
        import MXFP8_quantizer

        _package = MXFP8_quantizer.load_package()
    case = state["case"]
    op = case["op"]
    if op == "mxfp4":
        q, s = _package.quantize_mxfp4(state["x"])
        return {"values": _package.dequantize_mxfp4(q, s, TYPES[case["out"]]), "scales": s}
    if op == "gemm":
        return _package.mxfp4_gemm(state["a_q"], state["b_q"], state["a_s"], state["b_s"], TYPES[case["out"]])
    cache = _package.MXFP8Cache(*state["cache"])
    if op == "write":
        _package.cache_write(cache, state["k"], state["v"], state["slots"])
        return state["cache"]
    if op == "read":
        return _package.cache_read(cache, state["table"], state["starts"], state["total"], TYPES[case["out"]])
    out, lse = _package.cache_attention(state["q"], cache, state["table"], state["lengths"], return_lse=True)
    return {"out": out, "lse": lse}


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------
# what a pass cannot do without, and its value in 64 bits
# --------------------------------------------------------------------------

def work(case):
    op = case["op"]
    row = 1 + 1 / BLOCK                                   # bytes of a cached element with its share of the scale
    if op == "mxfp4":
        m, k = case["m"], _ceil(case["k"], BLOCK)
        # x in, values and scales out; the codes in between are not counted
        return {"bytes": m * (2 * case["k"] + k / BLOCK + k * BYTES[case["out"]]), "flops": 0}
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * k * (0.5 + 1 / BLOCK) + m * n * BYTES[case["out"]], "flops": 2 * m * n * k}
    if op == "write":
        return {"bytes": case["tokens"] * (8 + 2 * case["heads"] * case["dim"] * (2 + row)), "flops": 0}
    total = sum(_lengths(case))
    cached = 2 * total * case["heads"] * case["dim"] * row
    if op == "read":
        return {"bytes": cached + 2 * total * case["heads"] * case["dim"] * BYTES[case["out"]], "flops": 0}
    q = case["batch"] * case["heads"] * case["groups"] * case["dim"]
    return {"bytes": cached + 2 * q * 2, "flops": 4 * total * case["heads"] * case["groups"] * case["dim"]}


def _power64(byte):
    return torch.pow(torch.tensor(2.0, dtype=torch.float64, device=byte.device), byte.double() - 127)


def _rounded(y, bits, lowest, top):
    """y to the nearest value of `bits` explicit mantissa bits and exponents from `lowest`, ties to even, capped."""
    a = y.abs().clamp(min=2.0 ** lowest)
    step = torch.exp2(torch.floor(torch.log2(a)) - bits)
    return (torch.round(y / step) * step).clamp(-top, top)


def _mxfp8_exact(x):
    v = x.double().unflatten(-1, (-1, BLOCK))
    amax = v.abs().amax(-1)
    # the recipe's constants are the 32-bit neighbours of 1/448 and 1e-12, and its sum is held in 32 bits
    want = (amax * 0.002232142956927418708801269531 + 9.999999960041972002500187955e-13).float().double()
    e = torch.floor(torch.log2(want))
    e = e + (want > torch.exp2(e)).double()
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    return _rounded(v / torch.exp2(e)[..., None], 3, -6, 448.0).flatten(-2), (e + 127).to(torch.uint8)


def _rows64(pages, scales, table, b, length):
    """Sequence b's rows 0..length-1 in 64 bits: (length, heads, dim)."""
    page = pages.shape[2]
    which = table[b, : -(-length // page)].long()
    value = pages[which].double().unflatten(-1, (-1, BLOCK)) * _power64(scales[which])[..., None]
    return value.flatten(-2).transpose(1, 2).flatten(0, 1)[:length]


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "mxfp4":
        m, k = state["x"].shape
        v = torch.zeros((m, _ceil(k, BLOCK)), dtype=torch.float64, device="cuda")
        v[:, :k] = state["x"]
        v = v.view(m, -1, BLOCK)
        amax = v.abs().amax(-1)
        e = torch.floor(torch.log2(amax.clamp(min=2.0 ** -140))) - 2
        e = (e + (amax > 6 * torch.exp2(e)).double()).clamp(min=-127)
        e = torch.where(amax == 0, torch.zeros_like(e), e)
        scale = torch.exp2(e)[..., None]
        return {"values": (_rounded(v / scale, 1, 0, 6.0) * scale).view(m, -1), "scales": None}
    if op == "gemm":
        if case["m"] * case["n"] * case["k"] > 6e11:
            return None
        table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device="cuda")
        sides = []
        for name in ("a", "b"):
            q = state[name + "_q"]
            v = torch.empty((q.shape[0], case["k"]), dtype=torch.float64, device="cuda")
            v[:, 0::2] = table[(q % 16).long()]
            v[:, 1::2] = table[(q // 16).long()]
            s = state[name + "_s"][_chunk_index(q.shape[0], case["k"] // BLOCK, "cuda")]
            sides.append((v.view(q.shape[0], -1, BLOCK) * _power64(s)[..., None]).view(q.shape[0], -1))
        return sides[0] @ sides[1].t()
    if op == "write":
        cache = [t.double() if t.dtype == torch.float8_e4m3fn else None for t in state["cache"]]
        at = [i for i, s in enumerate(state["slots"].tolist()) if s >= 0]
        slot = state["slots"][at]
        for i, x in enumerate(("k", "v")):
            cache[i][slot // case["page"], :, slot % case["page"]] = _mxfp8_exact(state[x][at])[0]
        return tuple(cache)
    k_pages, v_pages, k_scales, v_scales = state["cache"]
    if op == "read":
        lens = (state["starts"][1:] - state["starts"][:-1]).tolist()
        return tuple(torch.cat([_rows64(p, s, state["table"], b, n) for b, n in enumerate(lens)])
                     for p, s in ((k_pages, k_scales), (v_pages, v_scales)))
    outs, lses = [], []
    for b, n in enumerate(state["lengths"].tolist()):
        q = state["q"][b].double().view(case["heads"], case["groups"], case["dim"])
        if n == 0:
            outs.append(torch.zeros_like(q))
            lses.append(torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda"))
            continue
        k = _rows64(k_pages, k_scales, state["table"], b, n)
        score = torch.einsum("hgd,lhd->hgl", q, k) * case["dim"] ** -0.5
        lses.append(torch.logsumexp(score, -1))
        p = torch.exp(score - lses[-1][..., None])
        outs.append(torch.einsum("hgl,lhd->hgd", p, _rows64(v_pages, v_scales, state["table"], b, n)))
    return {"out": torch.stack(outs).flatten(1, 2), "lse": torch.stack(lses).flatten(1)}
