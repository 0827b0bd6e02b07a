"""The MXFP4 oracle against hand-written cases and against brute force; runs without a GPU."""
import numpy as np

from oracle import mx


def test_known_block():
    x = np.zeros(32)
    x[:10] = [4.0, -0.25, 0.25, 0.75, 1.25, 2.5, 3.5, 5.0, 7.9, -0.0]
    codes, scale = mx.quantise(x)
    assert scale.tolist() == [127]                    # 7.9 lies in [4, 8): scale 1
    v = mx.values(codes, scale)
    assert v[:10].tolist() == [4.0, -0.0, 0.0, 1.0, 1.0, 2.0, 4.0, 4.0, 6.0, -0.0]
    assert np.signbit(v[1]) and np.signbit(v[9])
    assert (codes[0] & 15, codes[0] >> 4) == (6, 8)    # the lower half first


def test_ends_of_the_range():
    for x, byte in ((2.0**127 * 1.9, 252), (2.0**-126, 0), (2.0**-125, 0), (2.0**-124, 1), (2.0**-149, 0), (0.0, 0)):
        _, s = mx.quantise(np.full(32, x))
        assert s[0] == byte, x
    for bad in (np.inf, -np.inf, np.nan):
        x = np.ones(64)
        x[3] = bad
        codes, s = mx.quantise(x)
        assert s.tolist() == [255, 125] and (codes[:16] == 0).all()
        assert np.isnan(mx.values(codes, s)[:32]).all() and (mx.values(codes, s)[32:] == 1).all()


def test_nearest_and_ragged():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((40, 77)) * np.exp2(rng.integers(-20, 20, (40, 77)))
    codes, s = mx.quantise(x)
    assert codes.shape == (40, 48) and s.shape == (40, 3)
    v = mx.values(codes, s)
    assert (v[:, 77:] == 0).all()
    scale = np.repeat(np.exp2(s.astype(float) - 127), 32, axis=1)[:, :77]
    grid = np.concatenate([mx.GRID, -mx.GRID])
    best = np.abs(x[..., None] - grid * scale[..., None]).min(-1)
    assert (np.abs(x - v[:, :77]) == best).all()
    again = mx.quantise(v)
    assert (mx.values(*again) == v).all()             # values on the grid stay
