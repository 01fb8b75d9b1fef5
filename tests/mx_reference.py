"""MXFP4 restated in float64 on the host, from the format's definition: blocks of 32 along the last axis, one power-of-two
scale, e2m1 data.  Numpy only; every intermediate is exact (a division by a power of two and a rounding to a grid)."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """(codes uint8 0..15, scale bytes uint8) of a float64 array [..., K]."""
    b = np.asarray(x, dtype=np.float64).reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    m = np.abs(b).max(axis=-1)          # NaN where the block holds one
    bad = ~np.isfinite(m)
    _, e = np.frexp(np.where(bad | (m == 0), 1.0, m))
    byte = np.where(bad, 255, np.where(m == 0, 0, np.maximum(e - 1 - 2 + 127, 0))).astype(np.int64)
    t = np.abs(np.where(bad[..., None], 0.0, b)) * np.exp2(127.0 - np.where(bad, 127, byte))[..., None]
    # nearest of the grid, ties to the even code (the even ones are 0, 1, 2, 4: the values at even places)
    hi = np.clip(np.searchsorted(GRID, t, side="left"), 0, 7)
    lo = np.maximum(hi - 1, 0)
    dlo, dhi = t - GRID[lo], GRID[hi] - t
    code = np.where(dlo < dhi, lo, np.where(dlo > dhi, hi, np.where(lo % 2 == 0, lo, hi)))
    code = np.where(t >= 6.0, 7, code)
    sign = np.where(bad[..., None], False, np.signbit(b))
    return (code + 8 * sign).astype(np.uint8).reshape(x.shape), byte.astype(np.uint8)


def values(codes, scale_bytes):
    """float64 values of codes [..., K] under scale bytes [..., K / 32]."""
    c = codes.astype(np.int64)
    v = np.where(c >= 8, -1.0, 1.0) * GRID[c & 7]
    s = np.where(scale_bytes == 255, np.nan, np.exp2(scale_bytes.astype(np.float64) - 127.0))
    return v * np.repeat(s, 32, axis=-1)


def pack(codes):
    c = codes.reshape(-1, 2)
    return (c[:, 0] | (c[:, 1] << 4)).astype(np.uint8)


def unpack(packed, shape):
    return np.stack([packed & 15, packed >> 4], axis=-1).reshape(shape)
