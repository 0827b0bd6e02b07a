"""The gradient of the gated activation over every gate, with gradients and values whose products with the slope leave fp32's range one way or the other.

Bounds.  In fp32 the sigmoid s is off by (|g| + 16) 2^-23 of itself (the exponential's argument g log2(e) by 2^-24 of itself; exponential, sum and reciprocal by some roundings of
2^-23 each), the slope s (1 + g (1 - s)) by that of s (1 + |g|), and gradient, value and slope are multiplied with two roundings more, which the 16 hold.  The product of gradient and value below
2^-126 is off by 2^-150, and a slope is at most 1.1, so that a result is off by 2^-149 more at most.  A sigmoid below 2^-126 (g < -87.3) may be 0.  A result of 16 bits is rounded once, by half
a step.  Beyond |g| = 200 the slope is 1 or below 2^-280, in 64 bits as in 32."""
import pytest
import torch

import flux_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16 = torch.bfloat16, torch.float16


def exact(d, u, g):
    """Of the gate's gradient in 64 bits: the value, and what fp32 may be off."""
    near = g.clamp(-200, 200)
    e = torch.exp(-near.abs())
    s, rest = torch.where(near >= 0, 1, e) / (1 + e), torch.where(near >= 0, e, 1) / (1 + e)  # rest = 1 - s
    want = d * u * s * (1 + near * rest)
    slack = (d * u).abs() * s * (1 + near.abs()) * (near.abs() + 16) * 2.0**-23 + 2.0**-149
    return want, slack + torch.where(g < -87, (d * u * near).abs() * 2.0**-125, 0.0)


def check(got, want, slack):
    """Values beyond the type are infinite; within the bounds of its largest they may be either."""
    info = torch.finfo(got.dtype)
    off, bound = (got.double() - want).abs(), (want.abs() + slack) * info.eps / 2 + slack + info.tiny * info.eps / 2
    beyond = want.abs() + bound > info.max
    assert (off <= bound * 1.0000001)[~beyond].all(), f"off by {(off - bound)[~beyond].max().item():.3g} more than the bound"
    inf = want.abs() - bound > info.max * (1 + info.eps)
    assert (got[inf].double() == torch.copysign(torch.full_like(want[inf], float("inf")), want[inf])).all()


# Gradient and value: ordinary ones; a product of about 1 of factors far apart, either way; beyond fp32; below it.
BF16_PAIRS = [(0.7, 1.3), (1.7 * 2.0**-100, 1.1 * 2.0**100), (1.3 * 2.0**100, -1.9 * 2.0**-100), (2.0**-60, 1.5 * 2.0**80), (-(2.0**-120), 1.5 * 2.0**127), (1.0, 1.9 * 2.0**127),
              (1.5 * 2.0**99, 1.1 * 2.0**100), (1.5 * 2.0**127, 1.75 * 2.0**127), (1.9, -1.9 * 2.0**127), (2.0**-70, 1.5 * 2.0**-70), (1.5 * 2.0**-130, 2.0**10)]
F16_PAIRS = [(0.7, 1.3), (2.0**-24, 65504.0), (65504.0, 2.0**-24), (65504.0, 65504.0), (2.0**-24, 2.0**-24)]


@pytest.mark.parametrize("dtype,pair", [(BF16, p) for p in BF16_PAIRS] + [(F16, p) for p in F16_PAIRS])
def test_every_gate(dtype, pair):
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    g = x[torch.isfinite(x.float())].view(-1, 64).to(DEV)
    d, u = (torch.full_like(g, v) for v in pair)
    grad_input, _ = flux_amd.moe_swiglu_backward(d, torch.cat([g, u], 1))
    check(grad_input[:, :64], *exact(d.double(), u.double(), g.double()))


@pytest.mark.parametrize("d,u", [(1.5 * 2.0**-100, 2.0**100), (2.0**-60, 2.0**80), (1.0, 2.0**127), (2.0**100, 2.0**100)])
def test_gates_kept_in_8_bits(d, u):
    """The same from codes: gates that are values of e4m3, one scale to a half."""
    gates = torch.tensor([-80.0, -72.0, -60.0, -40.0, -30.0, -1.25, -0.5, 0.0, 0.5, 40.0, 88.0, 1.0] + [-52.0] * 20, dtype=BF16, device=DEV).repeat(3, 1)
    _, codes, scale = flux_amd.moe_swiglu_checkpoint(torch.cat([gates, torch.full_like(gates, u)], 1))
    grad = torch.full_like(gates, d)
    grad_input, _ = flux_amd.moe_swiglu_backward(grad, codes, scale)
    # (the greatest magnitude, 88, has a scale of 2^-2: multiples of 1/2048 up to 448 / 4 with four significant bits)
    kept = codes.view(torch.uint8).view(torch.float8_e4m3fn)[:, :32].float() * 2.0**-2
    assert scale.view(torch.uint8)[0, 0] == 125 and (kept - gates.float()).abs().max() <= 4
    check(grad_input[:, :32], *exact(grad.double(), torch.full_like(kept, u).double(), kept.double()))


def test_one_product_beyond_the_range_among_others():
    """Of a lane's eight values one alone takes the other order; infinities, zeros and NaN as the formula has them."""
    g = torch.full((1, 8), -30.0, dtype=BF16, device=DEV)
    d, u = torch.full_like(g, 2.0**-100), torch.full_like(g, 2.0**90)
    d[0, 3], u[0, 3] = 2.0**80, 2.0**80
    grad_input, _ = flux_amd.moe_swiglu_backward(d, torch.cat([g, u], 1))
    check(grad_input[:, :8], *exact(d.double(), u.double(), g.double()))
    inf = float("inf")
    d = torch.tensor([[inf, inf, 0.0, float("nan"), inf, 1.0, -inf, 0.0]], dtype=BF16, device=DEV)
    u = torch.tensor([[1.0, 0.0, inf, 1.0, inf, inf, 2.0, 5.0]], dtype=BF16, device=DEV)
    grad_input, _ = flux_amd.moe_swiglu_backward(d, torch.cat([g, u], 1))
    got = grad_input[0, :8].tolist()
    assert got[0] == -inf and got[4] == -inf and got[5] == -inf and got[6] == inf and got[7] == 0
    assert all(v != v for v in got[1:4])
