"""Float64 statements of the elementwise optimizer operators, in numpy: the AdamW step, and the 8-bit block format."""

import numpy as np


BLOCK = 256


def decay_factor(method, lr, wd):
    return {"decoupled": 1 - lr * wd, "independent": 1 - wd, "palm": 1 - lr * lr * wd, "l2": 1.0}[method]


def adamw(p, g, m, v, *, lr, betas, eps, wd, step, method="decoupled", scale=1.0):
    """New (p, m, v) and the magnitudes that rounding errors of p, m and v are relative to."""
    p, g, m, v = (np.asarray(x, dtype=np.float64) for x in (p, g, m, v))
    b1, b2 = betas
    g_mag = np.abs(g * scale)
    g = g * scale
    if method == "l2":
        g_mag = g_mag + np.abs(wd * p)
        g = g + wd * p
    m_mag = b1 * np.abs(m) + (1 - b1) * g_mag
    v_mag = b2 * v + (1 - b2) * g_mag**2
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    denom = np.sqrt(v / (1 - b2**step)) + eps
    size = lr / (1 - b1**step)
    new = p * decay_factor(method, lr, wd) - size * m / denom
    # v's own error moves the root by half of it, relative to v; v_mag >= v covers l2's cancellation
    with np.errstate(divide="ignore", invalid="ignore"):
        v_rel = np.where(v > 0, v_mag / np.maximum(v, 1e-300), 1.0)
    p_mag = np.abs(p) + size * (m_mag + np.abs(m) * (1 + v_rel)) / denom
    return (new, m, v), (p_mag, m_mag, v_mag)


def mix32(x):
    x = np.asarray(x, dtype=np.uint64)
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0x85EBCA6B)) & np.uint64(0xFFFFFFFF)
    x = ((x ^ (x >> np.uint64(13))) * np.uint64(0xC2B2AE35)) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def random_bits(numel, seed, tensor, step, signed, first=0):
    """The 16 random bits of elements ``first`` .. ``first + numel`` of a tensor."""
    key = mix32(mix32(mix32(seed) ^ np.uint64(tensor)) ^ np.uint64(step))
    r = mix32(key ^ (np.arange(first, first + numel, dtype=np.uint64) & np.uint64(0xFFFFFFFF)))
    return (r & np.uint64(0xFFFF)) if signed else (r >> np.uint64(16))


def _blocks(x):
    return np.pad(x, (0, -len(x) % BLOCK)).reshape(-1, BLOCK)


def quantize(x, signed, bits16=None):
    """Codes and exponent bytes of fp32 values, from the definition: four significant bits below the block's power of
    two, rounded up where the fraction cut off plus (r + 1/2) / 65536 (to nearest: plus 1/2) reaches one unit."""
    x = np.asarray(x, dtype=np.float64)
    bad = ~np.isfinite(x) | (False if signed else (x < 0))
    mag = np.where(bad, 0.0, np.abs(x))
    top = _blocks(mag).max(axis=1)
    exponent = np.maximum(np.frexp(top)[1] - 1, -126)  # of the largest power of two below
    exponent = np.where(top > 0, exponent, -126)
    t = np.ldexp(mag, -np.repeat(exponent, BLOCK)[: len(mag)])
    lowest = -13 if signed else -29
    e = np.where(t > 0, np.maximum(np.frexp(t)[1] - 1, lowest), lowest)
    u = 0.5 if bits16 is None else (np.asarray(bits16, dtype=np.float64) + 0.5) / 65536
    u = np.where(np.repeat(exponent, BLOCK)[: len(mag)] == 127, 0.0, u)
    units = np.floor(np.ldexp(t, 3 - e) + u)  # 8 .. 16 in a normal binade, 0 .. 8 below
    code = (e - lowest) * 8 + units  # the carry into the next binade is the next code
    if not signed:
        code = np.where((mag > 0) & (code == 0), 1, code)
    code = np.where(bad, 0x7F if signed else 0xFF, code).astype(np.int64)
    if signed:
        code = code + 128 * np.signbit(x)
    return code.astype(np.uint8), (exponent + 127).astype(np.uint8)


def dequantize(code, exponents, signed):
    c = np.asarray(code).astype(np.int64)
    sign = np.where(signed & (c >= 128), -1.0, 1.0)
    mag = c & 0x7F if signed else c
    e, mant = mag // 8, mag % 8
    top = 14 if signed else 30
    value = np.where(e > 0, np.ldexp(1 + mant / 8, e - top), np.ldexp(mant / 8, 1 - top))
    scale = np.ldexp(1.0, np.repeat(exponents.astype(np.int64), BLOCK)[: len(c)] - 127)
    return np.where(mag == (0x7F if signed else 0xFF), np.nan, sign * value * scale)


def join(p_bits, remainder):
    """fp32 masters of bf16 bit patterns and their remainders."""
    bits = (p_bits.astype(np.int64) << 16) + remainder.astype(np.int64)
    return (bits & 0xFFFFFFFF).astype(np.uint32).view(np.float32)
