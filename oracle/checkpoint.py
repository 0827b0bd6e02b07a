"""Activation checkpoints in 8 bits, in NumPy and from the definition: blocks of 32 values along the last axis share a power of two, a code is an e4m3 number.

Written in float64, in which every step is exact for 16-bit inputs; a test oracle, not part of the framework."""
import numpy as np

BLOCK = 32
# The magnitudes of e4m3 by code, 0 .. 448: subnormals in steps of 2^-9, then eight to each power of two.
GRID = np.array([c / 512.0 if c < 8 else np.exp2(c // 8 - 7.0) * (1 + c % 8 / 8) for c in range(127)])
_BORDERS = (GRID[1:] + GRID[:-1]) / 2  # halfway between neighbours: a tie
LARGEST = {"bf16": 1.875 * 2.0**127, "f16": 1.875 * 2.0**15}


def blocks(cols):
    return -(-cols // BLOCK)


def quantise(x, dtype):
    """x [..., cols] of 16-bit values -> (codes uint8 [..., cols], scales uint8 [..., blocks])."""
    x = np.asarray(x, dtype=np.float64)
    cols = x.shape[-1]
    x = np.pad(x, [(0, 0)] * (x.ndim - 1) + [(0, -cols % BLOCK)]).reshape(*x.shape[:-1], -1, BLOCK)
    bad = ~np.isfinite(x).all(-1)
    most = np.abs(np.where(bad[..., None], 0.0, x)).max(-1)
    byte = np.zeros(most.shape, dtype=np.int64)
    for b in range(248, -1, -1):                       # the least scale that 448 of reach the largest magnitude
        byte = np.where(most <= 448 * np.exp2(b - 127.0), b, byte)
    byte = np.where(bad, 255, byte)
    a = np.minimum(np.abs(np.where(bad[..., None], 0.0, x)), LARGEST[dtype]) * np.exp2(127.0 - np.where(bad, 127, byte))[..., None]
    low, high = np.searchsorted(_BORDERS, a, side="left"), np.searchsorted(_BORDERS, a, side="right")
    code = np.where(low % 2 == 0, low, high)           # they differ on a tie only: the even code
    code = np.where(np.signbit(x) & ~bad[..., None], code | 128, code).astype(np.uint8)
    return code.reshape(*code.shape[:-2], -1)[..., :cols], byte.astype(np.uint8)


def values(codes, scales):
    """The values of codes [..., cols] (no NaN among them), float64; NaN where the scale byte is 255."""
    v = GRID[np.minimum(codes & 127, 126)] * np.where(codes & 128, -1.0, 1.0)
    scale = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127.0))
    return v * np.repeat(scale, BLOCK, axis=-1)[..., :codes.shape[-1]]
