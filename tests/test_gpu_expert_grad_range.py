"""Gradients of the experts' products at the ends of the types: subnormal and largest values, and checkpoints whose scales are the least and the largest, by tiles and by pieces.

A sum of n products in fp32 is off by n 2^-23 of the sum of magnitudes (every product of 16-bit numbers is exact; the other factor keeps it in fp32's range); a result of 16 bits is rounded once.
In the matrix unit a subnormal counts as the least normal number for that: it adds products that are aligned by the sums of their factors' exponents, keeps 24 bits below the largest of
them, and a subnormal has the exponent of the least normal number though its leading bits are 0.  So 2^-23 is of max(|a|, tiny) max(|b|, tiny); alone in its sum every product is exact."""
import numpy as np
import pytest
import torch

import flux_amd
from oracle import checkpoint

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def signs(shape, dtype, seed, exponents):
    """Values of either sign, of all significands of the type, with exponents of a range."""
    g = torch.Generator().manual_seed(seed)
    e = torch.randint(exponents[0], exponents[1] + 1, shape, generator=g).double()
    return ((1 + torch.rand(*shape, generator=g).double()) * torch.exp2(e) * (torch.randint(0, 2, shape, generator=g) * 2 - 1)).to(dtype).to(DEV)


def close(got, want, slack):
    eps = torch.finfo(got.dtype).eps / 2 if got.dtype != F32 else 0.0
    bound = (want.abs() + slack) * eps + slack + torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    assert torch.isfinite(got).all() and ((got.double() - want).abs() <= bound * 1.0000001).all()


def size(t, dtype):
    """Magnitudes as the matrix unit aligns them: of values of a 16-bit type, in 64 bits."""
    return torch.where(t == 0, 0.0, t.abs().clamp(min=torch.finfo(dtype).tiny))


# (splits, n, k): by tiles, and by pieces
SIZES = [([9, 0, 40, 3, 33, 8, 1, 2], 1024, 1040), ([9, 0, 40], 72, 40), ([7, 12], 33, 45)]
# Exponents of the product's input (or weights) and of the gradient.
BF16_RANGES = [((-133, -127), (90, 110)), ((120, 126), (-110, -100)), ((-126, -100), (90, 100))]
F16_RANGES = [((-24, -15), (10, 14)), ((12, 14), (-24, -15))]
RANGES = [(BF16, *r) for r in BF16_RANGES] + [(F16, *r) for r in F16_RANGES]


@pytest.mark.parametrize("splits,n,k", SIZES)
@pytest.mark.parametrize("dtype,of_other,of_grad", RANGES)
@pytest.mark.parametrize("kept", [False, True])
def test_weights_at_the_ends_of_the_types(splits, n, k, dtype, of_other, of_grad, kept):
    rows = sum(splits)
    grad, x, scale = signs((rows, n), dtype, 1, of_grad), signs((rows, k), dtype, 2, of_other), None
    x64 = x.double()
    if kept:
        x, scale = flux_amd.moe_checkpoint(x)
        x64 = torch.from_numpy(checkpoint.values(x.view(torch.uint8).cpu().numpy(), scale.view(torch.uint8).cpu().numpy())).to(DEV)
        assert dtype == F16 or of_other[0] > -127 or (scale.view(torch.uint8) == 0).any()
    got = flux_amd.moe_wgrad(grad, x, torch.tensor(splits, dtype=torch.int32, device=DEV), scale, output_dtype=F32)
    at = 0
    for e, s in enumerate(splits):
        g, v = grad[at:at + s].double(), x64[at:at + s]
        close(got[e], g.t() @ v, (s * 2.0**-23 if s > 1 else 0.0) * (size(g, dtype).t() @ size(v, dtype)))
        at += s


@pytest.mark.parametrize("splits,n,k", [([9, 0, 300], 2056, 264), ([9, 0, 40], 72, 40), ([7, 12], 33, 45)])
@pytest.mark.parametrize("dtype,of_other,of_grad", RANGES[:4])
def test_inputs_at_the_ends_of_the_types(splits, n, k, dtype, of_other, of_grad):
    if dtype == F16:
        of_grad = (-6, -4)  # (the result is of 16 bits)
    elif of_other[1] > 0:
        of_grad = (-120, -115)
    grad, weight = signs((sum(splits), n), dtype, 1, of_grad), signs((len(splits), n, k), dtype, 2, of_other)
    got, at = flux_amd.moe_dgrad(grad, weight, torch.tensor(splits, dtype=torch.int32, device=DEV)), 0
    for e, s in enumerate(splits):
        g, w = grad[at:at + s].double(), weight[e].double()
        close(got[at:at + s], g @ w, n * 2.0**-23 * (size(g, dtype) @ size(w, dtype)))
        at += s


@pytest.mark.parametrize("n,k", [(1024, 1040), (72, 64)])
def test_every_scale_byte(n, k):
    """A checkpoint of the user's own making: every scale from 2^-127 to 2^126 with codes of magnitude 1, times gradients that bring the product to about 1."""
    rows = 256
    byte = torch.arange(254).clamp(max=253).tolist() + [127, 127]
    scale = torch.tensor(byte, dtype=torch.uint8).repeat(-(-k // 32), 1).t().contiguous().to(DEV).view(torch.float8_e8m0fnu)
    codes = torch.ones(rows, k).to(torch.float8_e4m3fn).to(DEV)
    e = torch.tensor(byte).double() - 127
    grad = torch.zeros(rows, n, dtype=BF16)
    grad[:, 0] = torch.exp2(-e.clamp(min=-126)).to(BF16)  # 1 each (the least scale: 1/2)
    for i in range(1, n):
        grad[(i * 7) % rows, i] = grad[(i * 7) % rows, 0]  # one row each: its scale alone
    got = flux_amd.moe_wgrad(grad.to(DEV), codes, torch.tensor([rows] + [0] * 7, dtype=torch.int32, device=DEV), scale, output_dtype=F32)[0].cpu()
    want = torch.ones(n)
    want[0] = 255.5
    want[1:] = torch.tensor([0.5 if byte[(i * 7) % rows] == 0 else 1.0 for i in range(1, n)])
    assert np.array_equal(got.numpy(), want.view(n, 1).expand(n, k).numpy())


@pytest.mark.parametrize("kept", [False, True])
def test_as_many_experts_as_there_may_be(kept):
    """1024 of them by tiles: whole tables, and tiles from the queues."""
    n, k, g = 264, 272, torch.Generator().manual_seed(1)
    splits = torch.randint(0, 9, (1024,), generator=g).tolist()
    splits[0], splits[1023] = 40, 33
    rows, at = sum(splits) + 3, torch.tensor([0] + splits).cumsum(0).tolist()
    on = torch.tensor(splits, dtype=torch.int32, device=DEV)
    grad, x, w, scale = signs((rows, n), BF16, 1, (-3, 0)), signs((rows, k), BF16, 2, (-3, 0)), signs((1024, n, k), BF16, 3, (-3, 0)), None
    x64 = x.double()
    if kept:
        x, scale = flux_amd.moe_checkpoint(x)
        x64 = torch.from_numpy(checkpoint.values(x.view(torch.uint8).cpu().numpy(), scale.view(torch.uint8).cpu().numpy())).to(DEV)
    dw, dx = flux_amd.moe_wgrad(grad, x, on, scale, output_dtype=F32), flux_amd.moe_dgrad(grad, w, on)
    for e in range(1024):
        g64, v = grad[at[e]:at[e + 1]].double(), x64[at[e]:at[e + 1]]
        close(dw[e], g64.t() @ v, max(splits) * 2.0**-23 * (g64.abs().t() @ v.abs()))
        if not kept:
            close(dx[at[e]:at[e + 1]], g64 @ w[e].double(), n * 2.0**-23 * (g64.abs() @ w[e].double().abs()))
    assert not dx[-3:].any()


WIDE = (1 << 22) - 8  # the most that tiles take
PLACES = [0, 1, 255, 256, 2097143, 2097152, WIDE - 257, WIDE - 8, WIDE - 1]


def test_the_widest_sum_of_tiles():
    """300 rows of the widest gradient: 256 of them are 2 GiB less 4 KiB.  Few values are not 0, so that the sums are short."""
    grad, w = torch.zeros(300, WIDE, dtype=BF16, device=DEV), torch.zeros(1, WIDE, 264, dtype=BF16, device=DEV)
    few, rows = signs((300, len(PLACES)), BF16, 1, (-3, 0)), signs((len(PLACES), 264), BF16, 2, (-3, 0))
    grad[:, PLACES], w[0, PLACES] = few, rows
    got = flux_amd.moe_dgrad(grad, w, torch.tensor([290], dtype=torch.int32, device=DEV))
    a, b = few[:290].double(), rows.double()
    close(got[:290], a @ b, len(PLACES) * 2.0**-23 * (a.abs() @ b.abs()))
    assert not got[290:].any()


@pytest.mark.parametrize("out", [BF16, F32])
def test_the_widest_results_of_tiles(out):
    """Rows of results of 8 or 16 MB: 256 of them end 8 KiB below 4 GiB in fp32."""
    grad, x = signs((40, 264), BF16, 1, (-3, 0)), signs((40, WIDE), BF16, 2, (-3, 0))
    total = torch.empty(1, 264, WIDE, dtype=out, device=DEV)
    got = flux_amd.moe_wgrad(grad, x, torch.tensor([37], dtype=torch.int32, device=DEV), output=total)[0]
    a = grad[:37].double()
    for c in range(0, WIDE, 1 << 20):
        b = x[:37, c:c + (1 << 20)].double()
        close(got[:, c:c + (1 << 20)], a.t() @ b, 37 * 2.0**-23 * (a.abs().t() @ b.abs()))
    old = got[:, PLACES].double()
    flux_amd.moe_wgrad(grad, x, torch.tensor([37], dtype=torch.int32, device=DEV), output=total, accumulate=True)
    b = x[:37, PLACES].double()
    close(got[:, PLACES], old + a.t() @ b, 37 * 2.0**-23 * (a.abs().t() @ b.abs()) + 2.0**-23 * (old.abs() + (a.t() @ b).abs()))


def test_the_tallest_results_of_tiles():
    """Experts of 16384 tiles along their rows, from the queues."""
    x, grad = signs((21, 136), BF16, 1, (-3, 0)), signs((21, WIDE), BF16, 2, (-3, 0))
    got = flux_amd.moe_wgrad(grad, x, torch.tensor([9, 12], dtype=torch.int32, device=DEV))
    for e, r in ((0, slice(0, 9)), (1, slice(9, 21))):
        a = x[r].double()
        for c in range(0, WIDE, 1 << 20):
            b = grad[r, c:c + (1 << 20)].double()
            close(got[e, c:c + (1 << 20)], b.t() @ a, 12 * 2.0**-23 * (b.abs().t() @ a.abs()))
