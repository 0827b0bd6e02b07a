"""The oracle of checkpoints in 8 bits against hand-written cases, torch's e4m3 and brute force; runs without a GPU."""
import numpy as np
import torch

from oracle import checkpoint


def test_grid_is_e4m3():
    want = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert (checkpoint.GRID == want).all()


def test_known_block():
    x = np.zeros(32)
    x[:8] = [448.0, -0.001, 17.0, 19.0, 2.0**-9, 2.0**-10, 3 * 2.0**-10, -0.0]
    codes, scale = checkpoint.quantise(x, "bf16")
    assert scale.tolist() == [127]
    v = checkpoint.values(codes, scale)
    assert v[:8].tolist() == [448.0, -2.0**-9 * 1.0 if 0.001 > 2.0**-10 else 0.0, 16.0, 20.0, 2.0**-9, 0.0, 2.0**-8, 0.0]
    assert np.signbit(v[7]) and codes[7] == 128
    assert checkpoint.quantise(np.full(32, 448.0001), "bf16")[1][0] == 128  # a scale further


def test_ends_of_the_range():
    for x, dtype, byte, value in ((1.9921875 * 2.0**127, "bf16", 247, 1.875 * 2.0**127), (65504.0, "f16", 135, 61440.0), (57344.0, "f16", 134, 57344.0),
                                  (2.0**-133, "bf16", 0, 2.0**-133), (2.0**-24, "f16", 95, 2.0**-24), (0.0, "bf16", 0, 0.0)):
        codes, s = checkpoint.quantise(np.full(3, x), dtype)
        assert s[0] == byte and checkpoint.values(codes, s)[0] == value, x
    for bad in (np.inf, -np.inf, np.nan):
        x = np.ones(64)
        x[3] = bad
        codes, s = checkpoint.quantise(x, "bf16")
        assert s.tolist() == [255, 119] and (codes[:32] == 0).all()
        assert np.isnan(checkpoint.values(codes, s)[:32]).all() and (checkpoint.values(codes, s)[32:] == 1).all()


def test_nearest_and_ragged():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((40, 77)) * np.exp2(rng.integers(-9, 9, (40, 77)))
    codes, s = checkpoint.quantise(x, "bf16")
    assert codes.shape == (40, 77) and s.shape == (40, 3)
    v = checkpoint.values(codes, s)
    scale = np.repeat(np.exp2(s.astype(float) - 127), 32, axis=1)[:, :77]
    grid = np.concatenate([checkpoint.GRID, -checkpoint.GRID])
    assert (np.abs(x - v) == np.abs(x[..., None] - grid * scale[..., None]).min(-1)).all()
    again = checkpoint.quantise(v, "bf16")
    assert (checkpoint.values(*again) == v).all()      # values on the grid stay


def test_values_are_values_of_the_type():
    """What a checkpoint of 16-bit values stands for has 16 bits itself: its use in a product rounds nothing."""
    for dtype, t in (("bf16", torch.bfloat16), ("f16", torch.float16)):
        x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(t)
        x = x[torch.isfinite(x.float())].double().numpy()
        for seed in range(4):
            codes, s = checkpoint.quantise(np.random.default_rng(seed).permutation(x), dtype)
            v = torch.from_numpy(checkpoint.values(codes, s))
            assert torch.equal(v, v.to(t).double())
