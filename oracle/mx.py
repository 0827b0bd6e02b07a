"""MXFP4 in NumPy, from the definition: blocks of 32 values along the last axis share a power of two, a value is the nearest of sixteen.

Written in float64, in which every step is exact for fp32 inputs; a test oracle, not part of the framework."""
import numpy as np

BLOCK = 32
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
_BORDERS = (GRID[1:] + GRID[:-1]) / 2  # halfway between neighbours: a tie


def blocks(cols):
    return -(-cols // BLOCK)


def quantise(x):
    """x [..., cols] -> (codes uint8 [..., 16 * blocks], scales uint8 [..., blocks])."""
    x = np.asarray(x, dtype=np.float64)
    pad = [(0, 0)] * (x.ndim - 1) + [(0, -x.shape[-1] % BLOCK)]
    x = np.pad(x, pad).reshape(*x.shape[:-1], -1, BLOCK)
    with np.errstate(invalid="ignore"):
        most = np.abs(x).max(-1)
    bad = ~np.isfinite(x).all(-1)
    _, e = np.frexp(np.where(bad, 1.0, most))       # most = m * 2^e, 0.5 <= m < 1
    byte = np.where(most == 0, 0, np.clip(e - 1 - 2 + 127, 0, 254))
    byte = np.where(bad, 255, byte)
    a = np.abs(np.where(bad[..., None], 0.0, x)) * np.exp2(127.0 - np.where(bad, 127, byte))[..., None]
    low, high = np.searchsorted(_BORDERS, a, side="left"), np.searchsorted(_BORDERS, a, side="right")
    code = np.where(low % 2 == 0, low, high)          # they differ on a tie only: the even code
    code = np.where(np.signbit(x) & ~bad[..., None], code | 8, code).astype(np.uint8)
    code = code.reshape(*code.shape[:-2], -1)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte.astype(np.uint8)


def values(codes, scales):
    """The values of packed codes, float64 [..., 32 * blocks]; NaN where the scale byte is 255."""
    nibble = np.stack([codes & 15, codes >> 4], axis=-1).reshape(*codes.shape[:-1], -1)
    v = GRID[nibble & 7] * np.where(nibble & 8, -1.0, 1.0)
    scale = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127.0))
    return v * np.repeat(scale, BLOCK, axis=-1)
