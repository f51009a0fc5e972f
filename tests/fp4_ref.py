"""MXFP4 in 64 bits (numpy), from the format's definition: the values that the
4-bit tests hold the kernels to."""

import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def bits_to_f64(bits, dtype):
    if dtype == "fp16":
        return bits.view(np.float16).astype(np.float64)
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def quantize(bits, dtype):
    """(m, k) 16-bit patterns -> (codes (m, kp) 0..15, scale bytes (m, kp/32)), kp = k rounded up to 32."""
    m, k = bits.shape
    kp = -(-k // 32) * 32
    x = np.zeros((m, kp))
    x[:, :k] = bits_to_f64(bits, dtype)
    blocks = x.reshape(m, kp // 32, 32)
    fine = np.isfinite(blocks).all(-1)
    v = np.where(fine[..., None], blocks, 0.0)
    amax = np.abs(v).max(-1)
    e = np.full(amax.shape, -127)
    while True:                                     # the smallest e >= -127 with amax <= 6 * 2^e
        low = amax > 6.0 * np.exp2(e.astype(np.float64))
        if not low.any():
            break
        e = e + low
    e = np.where(amax == 0, 0, e)
    y = v / np.exp2(e.astype(np.float64))[..., None]
    mag = np.abs(y)[..., None]
    dist = np.abs(mag - E2M1)
    near = dist.min(-1, keepdims=True)
    tie = dist == near                              # one code, or two neighbours: then the even one
    even = tie & (np.arange(8) % 2 == 0)
    code = np.where((tie.sum(-1) > 1), even.argmax(-1), tie.argmax(-1))
    code = code | (np.signbit(y) & fine[..., None]).astype(np.int64) << 3
    return code.reshape(m, kp).astype(np.uint8), np.where(fine, e + 127, 255).astype(np.uint8)


def values(codes, scale_bytes):
    v = E2M1[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.exp2(scale_bytes.astype(np.float64) - 127)
    s = np.where(scale_bytes == 255, np.nan, s)
    return v * np.repeat(s, 32, axis=1)


def pack_codes(codes):
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def scale_positions(rows, blocks):
    r, c = np.meshgrid(np.arange(rows), np.arange(blocks), indexing="ij")
    return ((r // 128) * (-(-blocks // 4)) + c // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + c % 4


def pack_scales(dense):
    rows, blocks = dense.shape
    out = np.zeros(-(-rows // 128) * 128 * -(-blocks // 4) * 4, np.uint8)
    out[scale_positions(rows, blocks)] = dense
    return out


def random_matrix(rng, rows, cols, spread=3):
    """Payload bytes, packed scales and f64 values of a random MXFP4 matrix."""
    codes = rng.integers(0, 16, (rows, cols)).astype(np.uint8)
    bytes_ = rng.integers(127 - spread, 128 + spread, (rows, cols // 32)).astype(np.uint8)
    return pack_codes(codes), pack_scales(bytes_), values(codes, bytes_)
