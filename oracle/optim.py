"""CPU restatement of the optimizer over a list of tensors: gradient norm, AdamW in Keras form, 8-bit state encoding.

`adamw` in 64 bits is the formula; `state32` follows the stored state's documented arithmetic (single fp32 operations) so
that the 8-bit codes can be compared exactly."""
import math

import numpy as np

BLOCK = 256


def padded(n):
    return -(-n // BLOCK) * BLOCK


def grad_norm(grads, max_norm):
    s = math.fsum(float((np.asarray(g, dtype=np.float64) ** 2).sum()) for g in grads)
    norm = math.sqrt(s) if s >= 0 and math.isfinite(s) else float("nan") if math.isnan(s) else float("inf")
    return norm, (min(1.0, max_norm / norm) if norm > 0 else 1.0) if math.isfinite(norm) else float("nan")


def alpha(lr, b1, b2, t):
    return lr * math.sqrt(1.0 - b2 ** t) / (1.0 - b1 ** t)


def adamw(p, g, m, v, t, lr, b1, b2, eps, wd, scale=1.0):
    """one step in 64 bits; returns p, m, v"""
    p, g, m, v = (np.asarray(a, dtype=np.float64) for a in (p, g, m, v))
    g = g * scale
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p * (1 - lr * wd) - alpha(lr, b1, b2, t) * m / (np.sqrt(v) + eps), m, v


def state32(g, m, v, b1, b2, scale=1.0):
    """the state's recursion in single fp32 operations, as it is stored"""
    f = np.float32
    g = np.asarray(g, dtype=f) * f(scale)
    m, v = np.asarray(m, dtype=f), np.asarray(v, dtype=f)
    return m + (g - m) * f(1 - b1), v + (g * g - v) * f(1 - b2)


def _hash(x):
    x = np.asarray(x, dtype=np.uint64) & np.uint64(0xFFFFFFFF)
    low = np.uint64(0xFFFFFFFF)
    x ^= x >> np.uint64(16)
    x = (x * np.uint64(0x7FEB352D)) & low
    x ^= x >> np.uint64(15)
    x = (x * np.uint64(0x846CA68B)) & low
    return x ^ (x >> np.uint64(16))


def draws(n, t, seed):
    """(m's, v's) 16-bit rounding numbers of state positions 0 .. n-1 at step t"""
    key = _hash(np.uint64(seed) ^ _hash(t))
    h = _hash(np.arange(n, dtype=np.uint64) ^ key)
    return (h & np.uint64(0xFFFF)).astype(np.float64), (h >> np.uint64(16)).astype(np.float64)


def encode(x, u, digits, smallest, top, floor_positive):
    """x (whole blocks) -> (values of the codes before the scale, scales): the block's power of two puts its maximum at or under
    1.75 * 2^top; a magnitude between two codes goes up where remainder + u / 65536 reaches 1"""
    b = np.asarray(x, dtype=np.float64).reshape(-1, BLOCK)
    big = np.abs(b).max(1)
    bad = ~np.isfinite(big)
    frac, e = np.frexp(np.where(bad | (big == 0), 1.0, big))
    e = np.where(big == 0, -126, np.maximum(e - 1 + (frac > 0.875) - top, -126))
    scale = np.ldexp(1.0, e)
    with np.errstate(invalid="ignore"):
        z = np.where(bad[:, None], 0.0, np.abs(b) / scale[:, None]).reshape(-1)
    unit = np.ldexp(1.0, smallest - 23)        # fp32 holds what is under the smallest normal code to this
    z = np.where(z < np.ldexp(1.0, smallest), np.rint(z / unit) * unit, z)
    _, k = np.frexp(np.where(z == 0, 1e-300, z))
    step = np.ldexp(1.0, np.maximum(k - 1, smallest) - digits)
    q = np.floor(z / step + u / 65536.0) * step
    if floor_positive:
        q = np.where((q == 0) & (b.reshape(-1) > 0) & ~np.repeat(bad, BLOCK), np.ldexp(1.0, smallest - digits), q)
    return np.where(np.signbit(b.reshape(-1)), -q, q), np.where(bad, np.nan, scale)


def encode_m(x, u):
    return encode(x, u, 3, -6, 8, False)


def encode_v(x, u):
    return encode(x, u, 2, -14, 15, True)
