"""CPU restatement of 4-bit microscaled matrices (blocks of 32, E2M1 codes, E8M0 scales) in 64 bits."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """x (R, C) -> (codes uint8 (R, 32 blocks) with the sign in bit 3, scale bytes uint8 (R, blocks))"""
    x = np.asarray(x, dtype=np.float64)
    r, c = x.shape
    b = np.pad(x, ((0, 0), (0, -c % 32))).reshape(r, -1, 32)
    big = np.abs(b).max(2)
    bad = ~np.isfinite(big)
    frac, e = np.frexp(np.where(bad | (big == 0), 1.0, big))
    byte = np.clip(e - 1 - 2 + (frac > 0.875) + 127, 0, 254)
    byte = np.where(bad, 255, np.where(big == 0, 0, byte))
    with np.errstate(invalid="ignore", over="ignore"):
        a = np.where(bad[..., None], 0.0, np.abs(b) / np.ldexp(1.0, byte - 127)[..., None])
    # nearest grid value, ties to the even code
    d = np.abs(a[..., None] - GRID)
    near = d.min(-1, keepdims=True)
    tied = d == near
    first, last = tied.argmax(-1), 7 - tied[..., ::-1].argmax(-1)
    code = np.where(first % 2 == 0, first, last)
    code = np.where(bad[..., None], 0, code + 8 * np.signbit(b))
    return code.reshape(r, -1).astype(np.uint8), byte.astype(np.uint8)


def values(codes, scales, cols):
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    v = np.where(codes >= 8, -1.0, 1.0) * GRID[codes & 7]
    return (v.reshape(codes.shape[0], -1, 32) * s[..., None]).reshape(codes.shape[0], -1)[:, :cols]


def pack(codes):
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def unpack(packed):
    return np.stack([packed & 15, packed >> 4], 2).reshape(packed.shape[0], -1)


def round_trip(x):
    return values(*quantize(x), x.shape[1])
