"""The gradients of the grouped product, activation checkpoints in 8 bits and the layers made of them, against the formulas in 64 bits.

Bounds.  A sum of n products of 16-bit numbers in fp32: every product is exact, every addition is off by at most 2^-23 of the sum of magnitudes (truncation;
2^-24 if rounded), so n * 2^-23 of that in all; a result of 16 bits is rounded once more, half a step of the value.  silu: the exponential's argument g
log2(e) is off by 2^-24 of itself, which is |g| 2^-24 of the result, and exponential, sum, reciprocal and the products add some roundings of 2^-23 each: (|g| + 16)
2^-23 of the factors' magnitudes; a reciprocal below 2^-126 may be 0."""
import numpy as np
import pytest
import torch

import flux_amd
from flux_amd import capi
from oracle import checkpoint

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAME = {BF16: "bf16", F16: "f16"}


def data(shape, dtype, seed, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(DEV)


def counts(splits):
    return torch.tensor(splits, dtype=torch.int32, device=DEV)


def close(got, want, slack):
    """slack: what fp32 inside may be off."""
    assert got.shape == want.shape
    eps = torch.finfo(got.dtype).eps / 2 if got.dtype != F32 else 0.0
    bound = (want.abs() + slack) * eps + slack + torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    assert torch.isfinite(got).all()
    off = (got.double() - want).abs()
    assert (off <= bound * 1.0000001).all(), f"off by {(off - bound).max().item():.3g} more than the bound"


def ranges(splits, rows):
    """(expert, its rows), as the kernels see the counts."""
    at = 0
    for e, s in enumerate(splits):
        end = min(rows, at + max(0, s))
        yield e, slice(at, end)
        at = end


def want_dgrad(grad, weight, splits):
    out = torch.zeros(grad.shape[0], weight.shape[2], dtype=torch.float64, device=DEV)
    for e, r in ranges(splits, grad.shape[0]):
        out[r] = grad[r].double() @ weight[e].double()
    return out


def want_wgrad(grad, x, splits):
    out = torch.zeros(len(splits), grad.shape[1], x.shape[1], dtype=torch.float64, device=DEV)
    for e, r in ranges(splits, grad.shape[0]):
        out[e] = grad[r].double().t() @ x[r].double()
    return out


def values(codes, scale):
    return torch.from_numpy(checkpoint.values(codes.view(torch.uint8).cpu().numpy(), scale.view(torch.uint8).cpu().numpy())).to(DEV)


# (splits, rows behind them, n, k)
PRODUCTS = [([1], 0, 8, 8), ([0, 3, 0], 2, 16, 24), ([5, 0, 129, 64], 0, 128, 128), ([127, 1, 128], 5, 136, 264), ([33], 0, 1, 1), ([40, 7], 3, 31, 45),
            ([300, 0, 17], 130, 520, 72), ([2, 2, 2, 2, 2, 2, 2, 2], 0, 1024, 512), ([600, 500], 0, 257, 130), ([4000], 9, 64, 96), ([0, 0], 7, 64, 64),
            ([257, 511, 256, 1], 0, 768, 1288), ([70] * 70, 1, 64, 40), ([31, 32, 33, 65, 95], 0, 512, 256), ([2, -5, 30], 4, 72, 200)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("splits,rest,n,k", PRODUCTS)
def test_dgrad(splits, rest, n, k, dtype):
    print(f"[case] dgrad {splits[:6]} {rest} {n} {k} {dtype}", flush=True)
    rows = sum(max(0, s) for s in splits) + rest
    grad, weight = data((rows, n), dtype, 1), data((len(splits), n, k), dtype, 2)
    grad[rows - rest:] = float("nan")  # rows of no expert are not used
    got = flux_amd.moe_dgrad(grad, weight, counts(splits))
    close(got, want_dgrad(grad, weight, splits), n * 2.0**-23 * want_dgrad(grad.abs(), weight.abs(), splits))
    assert (got[rows - rest:] == 0).all()
    assert torch.equal(got, capi.moe_dgrad(grad, weight, counts(splits)))
    assert torch.equal(got, flux_amd.moe_dgrad(grad, weight, torch.tensor(splits, dtype=torch.int32)))


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("out", ["same", F32])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("splits,rest,n,k", PRODUCTS)
def test_wgrad(splits, rest, n, k, dtype, out, kept):
    print(f"[case] wgrad {splits[:6]} {rest} {n} {k} {dtype} {out} {kept}", flush=True)
    rows = sum(max(0, s) for s in splits) + rest
    grad, x, scale = data((rows, n), dtype, 3), data((rows, k), dtype, 4), None
    grad[rows - rest:] = x[rows - rest:] = float("nan")
    x[:1] *= 100  # blocks of rows with scales far from each other
    if kept:
        x, scale = flux_amd.moe_checkpoint(x)
        x64 = values(x, scale)
    else:
        x64 = x.double()
    out = dtype if out == "same" else out
    got = flux_amd.moe_wgrad(grad, x, counts(splits), input_scale=scale, output_dtype=out)
    assert got.dtype == out
    want = want_wgrad(grad, x64, splits)
    slack = max(max(splits), 1) * 2.0**-23 * want_wgrad(grad.abs(), x64.abs(), splits)
    close(got, want, slack)
    assert torch.equal(got, capi.moe_wgrad(grad, x, counts(splits), scale, out))
    # added to what is there: one more rounding of the sum, and of the result
    old = data(got.shape, out, 5)
    total = old.clone()
    version = total._version
    assert flux_amd.moe_wgrad(grad, x, counts(splits), input_scale=scale, output=total, accumulate=True) is not None and total._version > version
    close(total, old.double() + want, slack + 2.0**-23 * (old.double().abs() + want.abs()))
    flux_amd.moe_wgrad(grad, x, counts(splits), input_scale=scale, output=total)
    assert torch.equal(total, got)


# Sums of every length around the steps of the tiles, widths that end anywhere in them, one and several tiles to a workgroup, and few tiles with long sums, which are
# cut.  The first of them are small for the weights' gradient (pieces of 128 x 128), and those with n below 2048 for the input's.
TILES = [([224, 255, 256, 257, 287, 288, 289, 320, 33], 1, 96, 48), ([1000, 31, 513], 0, 776, 528), ([s for s in range(0, 40)], 3, 264, 272),
         ([224, 255, 256, 257, 287, 288, 289, 320, 33, 0, 1] * 7, 1, 96, 48), ([40, 31, 70] * 14, 0, 776, 528), ([96, 500], 7, 2056, 2064), ([3000, 2001], 5, 1544, 1288),
         ([640, 0, 700], 40, 2048, 264), ([5, 0, 40, 129, 1], 2, 2056, 136), ([300, 250, 0, 600], 0, 2072, 72), ([257, 1, 255], 9, 4104, 256), ([9, 9], 300, 2064, 512)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("splits,rest,n,k", TILES)
def test_tiles(splits, rest, n, k, dtype):
    print(f"[case] tiles {splits[:6]} {rest} {n} {k} {dtype}", flush=True)
    rows = sum(splits) + rest
    grad, x, weight = data((rows, n), dtype, 3), data((rows, k), dtype, 4), data((len(splits), n, k), dtype, 5)
    grad[rows - rest:] = x[rows - rest:] = float("nan")  # rows of no expert are not used
    close(flux_amd.moe_dgrad(grad, weight, counts(splits)), want_dgrad(grad, weight, splits), n * 2.0**-23 * want_dgrad(grad.abs(), weight.abs(), splits))
    codes, scale = flux_amd.moe_checkpoint(x)
    for given, its_scale, x64 in ((x, None, x.double()), (codes, scale, values(codes, scale))):
        want, slack = want_wgrad(grad, x64, splits), max(splits) * 2.0**-23 * want_wgrad(grad.abs(), x64.abs(), splits)
        for out in (dtype, F32):
            got = flux_amd.moe_wgrad(grad, given, counts(splits), its_scale, output_dtype=out)
            close(got, want, slack)
            total = torch.ones_like(got)
            flux_amd.moe_wgrad(grad, given, counts(splits), its_scale, output=total, accumulate=True)
            close(total, want + 1, slack + 2.0**-23 * (1 + want.abs()))


@pytest.mark.parametrize("experts", [60, 150])
def test_many_tiles_to_a_workgroup(experts):
    """Thousands of tiles, of which neighbours differ in length, each against the tile's own call."""
    n, k = 1024, 1040
    g = torch.Generator().manual_seed(experts)
    splits = torch.randint(0, 90, (experts,), generator=g).tolist()
    rows = sum(splits) + 11
    grad, x, w = data((rows, n), BF16, 1), data((rows, k), BF16, 2), data((experts, n, k), BF16, 3)
    codes, scale = flux_amd.moe_checkpoint(x)
    for given, its_scale, x64 in ((x, None, x.double()), (codes, scale, values(codes, scale))):
        want, slack = want_wgrad(grad, x64, splits), 90 * 2.0**-23 * want_wgrad(grad.abs(), x64.abs(), splits)
        for out in (BF16, F32):
            close(flux_amd.moe_wgrad(grad, given, counts(splits), its_scale, output_dtype=out), want, slack)
    big = [s * 9 for s in splits]
    grad = data((sum(big) + 5, n), BF16, 4)
    close(flux_amd.moe_dgrad(grad, w, counts(big)), want_dgrad(grad, w, big), n * 2.0**-23 * want_dgrad(grad.abs(), w.abs(), big))


def test_counts_past_the_rows():
    """What the counts have past the rows does not exist; sums of them overflow nothing."""
    grad, x, w = data((50, 64), BF16, 1), data((50, 40), BF16, 2), data((3, 64, 40), BF16, 3)
    for splits in ([20, 2**31 - 1, 2**31 - 1], [60, 1, 1], [-(2**31), 50, 7]):
        close(flux_amd.moe_dgrad(grad, w, counts(splits)), want_dgrad(grad, w, splits), 64 * 2.0**-23 * want_dgrad(grad.abs(), w.abs(), splits))
        close(flux_amd.moe_wgrad(grad, x, counts(splits)), want_wgrad(grad, x, splits), 50 * 2.0**-23 * want_wgrad(grad.abs(), x.abs(), splits))
    many = [0] * 1024
    many[0] = many[1000] = 25
    w = data((1024, 64, 8), BF16, 4)
    close(flux_amd.moe_dgrad(grad, w, counts(many)), want_dgrad(grad, w, many), 64 * 2.0**-23 * want_dgrad(grad.abs(), w.abs(), many))
    close(flux_amd.moe_wgrad(grad, x, counts(many)), want_wgrad(grad, x, many), 50 * 2.0**-23 * want_wgrad(grad.abs(), x.abs(), many))


@pytest.mark.parametrize("offset", [1, 4])
@pytest.mark.parametrize("n,k", [(128, 256), (264, 320)])
def test_operands_at_any_element(offset, n, k):
    """Slices of larger buffers: the products' sums may run in another order, the results hold the same bounds."""
    splits = [70, 0, 61]

    def at(t):
        flat = torch.zeros(t.numel() + offset, dtype=t.dtype, device=DEV)
        flat[offset:] = t.flatten()
        return flat[offset:].view(t.shape)

    grad, x, w = (at(data(s, BF16, i)) for i, s in enumerate([(131, n), (131, k), (3, n, k)]))
    s = at(counts(splits))
    close(flux_amd.moe_dgrad(grad, w, s), want_dgrad(grad, w, splits), n * 2.0**-23 * want_dgrad(grad.abs(), w.abs(), splits))
    close(flux_amd.moe_wgrad(grad, x, s), want_wgrad(grad, x, splits), 70 * 2.0**-23 * want_wgrad(grad.abs(), x.abs(), splits))
    codes, scale = flux_amd.moe_checkpoint(x)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip((codes, scale), flux_amd.moe_checkpoint(x.clone())))
    got = flux_amd.moe_wgrad(grad, at(codes.view(torch.uint8)).view(codes.dtype), s, at(scale.view(torch.uint8)).view(scale.dtype))
    x64 = values(codes, scale)
    close(got, want_wgrad(grad, x64, splits), 70 * 2.0**-23 * want_wgrad(grad.abs(), x64.abs(), splits))


def test_infinities_stay_in_their_rows_and_experts():
    splits = [40, 33]
    grad, x, w = data((80, 72), BF16, 1), data((80, 64), BF16, 2), data((2, 72, 64), BF16, 3)
    grad[3, 7], x[50, 9], w[1, 5, 6] = float("inf"), float("nan"), float("-inf")
    dx, dw = flux_amd.moe_dgrad(grad, w, counts(splits)), flux_amd.moe_wgrad(grad, x, counts(splits))
    bad = ~torch.isfinite(dx)
    assert bad[3].all() and bad[40:73, 6].all()
    bad[3] = bad[40:73, 6] = False
    assert not bad.any()
    bad = ~torch.isfinite(dw)
    assert bad[0, 7].all() and bad[1, :, 9].all()
    bad[0, 7] = bad[1, :, 9] = False
    assert not bad.any()
    codes, scale = flux_amd.moe_checkpoint(x)  # a block of them is NaN
    dw = flux_amd.moe_wgrad(torch.ones_like(grad), codes, counts(splits), scale)
    assert torch.isnan(dw[1, :, :32]).all() and torch.isfinite(dw[0]).all() and torch.isfinite(dw[1, :, 32:]).all()


def test_infinities_in_the_steps_of_tiles():
    """The same by tiles: steps of which the next expert's rows and W's are no part, rows and columns that a tile does not have."""
    splits, n, k = [40, 33, 0, 70] * 8, 2056, 264
    grad, w = data((sum(splits) + 3, n), BF16, 1), data((len(splits), n, k), BF16, 2)
    grad[40], w[3, 5, 6], grad[-3:] = float("inf"), float("-inf"), float("nan")
    bad = ~torch.isfinite(flux_amd.moe_dgrad(grad, w, counts(splits)))
    assert bad[40].all() and bad[73:143, 6].all()
    bad[40] = bad[73:143, 6] = False
    assert not bad.any()
    n, k = 1032, 528
    grad, x = data((sum(splits) + 3, n), BF16, 3), data((sum(splits) + 3, k), BF16, 4)
    grad[40, 1031], x[72, 527], grad[-3:], x[-3:] = float("inf"), float("nan"), float("nan"), float("inf")
    bad = ~torch.isfinite(flux_amd.moe_wgrad(grad, x, counts(splits)))
    assert bad[1, 1031].all() and bad[1, :, 527].all()
    bad[1, 1031] = bad[1, :, 527] = False
    assert not bad.any()
    codes, scale = flux_amd.moe_checkpoint(x)
    bad = ~torch.isfinite(flux_amd.moe_wgrad(grad, codes, counts(splits), scale))
    assert bad[1, 1031].all() and bad[1, :, 512:].all()
    bad[1, 1031] = bad[1, :, 512:] = False
    assert not bad.any()


def test_offsets_past_32_bits():
    """Operands and results of more than 4 GiB."""
    g = torch.Generator(DEV).manual_seed(1)
    rows, n, k, splits = 700000, 4096, 64, [100, 699000, 800]  # 5.7 GB of gradients
    grad = torch.empty(rows, n, dtype=BF16, device=DEV)
    for r in range(0, rows, 100000):
        grad[r:r + 100000] = torch.randn(100000, n, generator=g, device=DEV).to(BF16)
    x, w = torch.randn(rows, k, generator=g, device=DEV).to(BF16), torch.randn(3, n, k, generator=g, device=DEV).to(BF16)
    got = flux_amd.moe_dgrad(grad, w, counts(splits))
    probe = torch.cat([torch.tensor([0, 99, 100, 699099, 699100, 699899, 699900]), torch.randint(0, rows, (50,))]).to(DEV)
    e = (probe >= 100).long() + (probe >= 699100).long()
    want = torch.stack([grad[r].double() @ w[i].double() if r < 699900 else torch.zeros(k, dtype=torch.float64, device=DEV) for r, i in zip(probe.tolist(), e.tolist())])
    close(got[probe], want, 2.0**-10 * n**0.5)
    got = flux_amd.moe_wgrad(grad, x, counts(splits), output_dtype=F32)
    cols = torch.tensor([0, 1, 2047, 4095], device=DEV)
    part = grad[:, cols].double()
    want = want_wgrad(part, x, splits)
    # (the worst case of so long a sum allows anything: sums of signs at random stay within 2^-23 times a few hundred of the magnitudes' root)
    assert ((got[:, cols].double() - want).abs() <= 1e-5 * want_wgrad(part.abs(), x.abs(), splits)).all()


def test_results_past_32_bits():
    """2.5 10^9 weights; most experts have no rows."""
    splits = [0] * 150
    splits[0], splits[149] = 5, 40
    grad, x = data((45, 4096), BF16, 1), data((45, 4096), BF16, 2)
    got = flux_amd.moe_wgrad(grad, x, counts(splits))
    for e, r in ((0, slice(0, 5)), (149, slice(5, 45))):
        close(got[e], grad[r].double().t() @ x[r].double(), 40 * 2.0**-23 * (grad[r].double().abs().t() @ x[r].double().abs()))
    assert not got[1:149].any()


# ---- checkpoints and the gated activation ---------------------------------------------------------------------------


ROWS = [(1, 1), (3, 31), (5, 33), (2, 64), (129, 2047), (64, 4096), (7, 20000), (1000, 96), (3, 8), (300, 1407)]


def same_kept(codes, scale, x):
    want_codes, want_scale = checkpoint.quantise(x.double().cpu().numpy(), NAME[x.dtype])
    assert np.array_equal(scale.view(torch.uint8).cpu().numpy(), want_scale)
    assert np.array_equal(codes.view(torch.uint8).cpu().numpy(), want_codes)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,cols", ROWS)
def test_checkpoint(rows, cols, dtype):
    x = data((rows, cols), dtype, cols)
    x[:, ::7] *= 30
    codes, scale = flux_amd.moe_checkpoint(x)
    assert codes.dtype == torch.float8_e4m3fn and scale.dtype == torch.float8_e8m0fnu
    same_kept(codes, scale, x)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip((codes, scale), capi.checkpoint_e4m3(x)))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_checkpoint_of_every_value(dtype):
    """All 65536 patterns beside values of their own size, smaller ones and larger ones; and alone, with zeros."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    alone = torch.zeros(65536, 32, dtype=dtype)
    alone[:, 5] = x
    finite = x[torch.isfinite(x.float())]
    sorted_ = torch.cat([finite, finite[: -finite.numel() % 32]]).sort().values.view(-1, 32)
    mixed = finite[torch.randperm(finite.numel(), generator=torch.Generator().manual_seed(1))][: finite.numel() // 64 * 64].view(-1, 64)
    for t in (alone, sorted_, mixed, x.view(-1, 256)):
        t = t.contiguous().to(DEV)
        same_kept(*flux_amd.moe_checkpoint(t), t)


def silu_slack(g):
    return (g.abs().double() + 16) * 2.0**-23


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,cols", ROWS)
def test_swiglu(rows, cols, dtype):
    x = data((rows, 2 * cols), dtype, cols + 1, 3.0)
    x[0, 0], x[-1, cols - 1] = 30.0, -30.0
    g, u = x[:, :cols].double(), x[:, cols:].double()
    want = torch.nn.functional.silu(g) * u
    out, codes, scale = flux_amd.moe_swiglu_checkpoint(x)
    close(out, want, want.abs() * silu_slack(g))
    assert torch.equal(out, flux_amd.moe_swiglu(x))
    kb = -(-cols // 32)
    assert scale.shape == (rows, 2 * kb)
    for h, half in enumerate((x[:, :cols], x[:, cols:])):
        same_kept(codes.view(torch.uint8)[:, h * cols:(h + 1) * cols], scale.view(torch.uint8)[:, h * kb:(h + 1) * kb], half)


def want_swiglu_backward(grad, g, u):
    """The gradient in 64 bits, and what fp32 may be off."""
    s = torch.sigmoid(g)
    silu = g * s
    slope = s * (1 + g * (1 - s))
    want = torch.cat([grad * u * slope, grad * silu], 1)
    # (1 - s is off by 2^-23 of 1, where it may be far smaller)
    slack = torch.cat([(grad * u * s).abs() * (1 + g.abs()), (grad * silu).abs()], 1) * silu_slack(g).repeat(1, 2)
    return want, slack + torch.cat([(grad * u * g).abs(), (grad * g).abs()], 1) * 2.0**-125, silu * u, (silu * u).abs() * silu_slack(g) + (g * u).abs() * 2.0**-125


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,cols", ROWS)
def test_swiglu_backward(rows, cols, dtype, kept):
    x, grad, scale = data((rows, 2 * cols), dtype, cols + 2, 3.0), data((rows, cols), dtype, cols + 3), None
    x[0, 0], x[-1, cols - 1] = 90.0, -90.0
    g, u = x[:, :cols].double(), x[:, cols:].double()
    if kept:
        _, x, scale = flux_amd.moe_swiglu_checkpoint(x)
        kb = -(-cols // 32)
        byte = scale.view(torch.uint8)
        g, u = values(x[:, :cols], byte[:, :kb]), values(x[:, cols:], byte[:, kb:])
    grad_input, out = flux_amd.moe_swiglu_backward(grad, x, scale)
    want, slack, want_out, out_slack = want_swiglu_backward(grad.double(), g, u)
    close(grad_input, want, slack)
    close(out, want_out, out_slack)


def test_gradient_of_a_closed_gate():
    """The gate's slope is 0 before the product of gradient and value, which alone is beyond fp32."""
    gated = torch.tensor([[-200.0] * 8 + [1e30] * 8], dtype=BF16, device=DEV)
    grad_input, out = flux_amd.moe_swiglu_backward(torch.full((1, 8), 1e30, dtype=BF16, device=DEV), gated)
    assert not grad_input[:, :8].any() and not grad_input[:, 8:].any() and not out.any()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gate_of_every_value(dtype):
    """Finite gates of any size give finite results where the product is one; infinities and NaN give what torch's silu gives."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype).view(-1, 64).to(DEV)
    gated = torch.cat([x, torch.ones_like(x)], 1)
    out = flux_amd.moe_swiglu(gated)
    finite = torch.isfinite(x.float())
    want = torch.nn.functional.silu(x[finite].double())
    eps, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    assert ((out[finite].double() - want).abs() <= want.abs() * (eps + silu_slack(x[finite].clamp(-1e4, 1e4)) * 1.01) + x[finite].double().abs() * 2.0**-125 + tiny).all()
    inf = x == float("inf")
    assert (out[inf] == float("inf")).all() and torch.isnan(out[torch.isnan(x) | (x == float("-inf"))]).all()
    grad_input, _ = flux_amd.moe_swiglu_backward(torch.ones_like(x), gated)
    assert torch.isfinite(grad_input[:, :64][finite]).all() and torch.isfinite(grad_input[:, 64:][finite]).all()


def test_many_rows_and_more_bytes_than_32_bits():
    rows, cols = 200000, 8192  # 6.5 GB of gated rows
    g = torch.Generator(DEV).manual_seed(2)
    x = torch.empty(rows, 2 * cols, dtype=BF16, device=DEV)
    for r in range(0, rows, 20000):
        x[r:r + 20000] = torch.randn(20000, 2 * cols, generator=g, device=DEV).to(BF16)
    out, codes, scale = flux_amd.moe_swiglu_checkpoint(x)
    probe = torch.tensor([0, 1, 99999, 131072, 199999], device=DEV)
    few = x[probe]
    a, b, c = flux_amd.moe_swiglu_checkpoint(few)
    assert torch.equal(out[probe], a) and torch.equal(codes.view(torch.uint8)[probe], b.view(torch.uint8))
    assert torch.equal(scale.view(torch.uint8)[probe], c.view(torch.uint8))
    grad_input, again = flux_amd.moe_swiglu_backward(out, codes, scale)
    a, b = flux_amd.moe_swiglu_backward(out[probe], b, c)
    assert torch.equal(grad_input[probe], a) and torch.equal(again[probe], b)


# ---- layers -----------------------------------------------------------------------------------------------------


def mlp64(x, w1, w2, splits):
    out = torch.zeros(x.shape[0], w2.shape[1], dtype=torch.float64, device=DEV)
    for e, r in ranges(splits, x.shape[0]):
        h = x[r] @ w1[e].t()
        f = h.shape[1] // 2
        out[r] = (torch.nn.functional.silu(h[:, :f]) * h[:, f:]) @ w2[e].t()
    return out


def mlp_operands(splits, rest, hidden, ffn, dtype, seed=1):
    rows = sum(splits) + rest
    return (data((rows, hidden), dtype, seed).requires_grad_(), data((len(splits), 2 * ffn, hidden), dtype, seed + 1, hidden**-0.5).requires_grad_(),
            data((len(splits), hidden, ffn), dtype, seed + 2, ffn**-0.5).requires_grad_())


def relative(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("ckpt", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("splits,rest,hidden,ffn", [([30, 0, 65], 4, 128, 96), ([300, 200, 7, 128], 0, 256, 320), ([9, 17], 2, 40, 24)])
def test_mlp_gradients(splits, rest, hidden, ffn, dtype, ckpt):
    """Every tensor between the products is rounded once (eps / 2), a checkpoint's value by 2^-4 of itself or less (2^-4 / sqrt(3) in the mean): a result's 2-norm is off by some
    of these roundings in a row, each scaled by factors around one (silu's slope and curvature); four times the roundings of the longest chain bound them."""
    x, w1, w2 = mlp_operands(splits, rest, hidden, ffn, dtype)
    out = flux_amd.moe_mlp(x, w1, w2, counts(splits), checkpoint=ckpt)
    up = data(out.shape, dtype, 9)
    out.backward(up)
    x64, a64, b64 = (t.detach().double().requires_grad_() for t in (x, w1, w2))
    want = mlp64(x64, a64, b64, splits)
    want.backward(up.double())
    half = torch.finfo(dtype).eps / 2
    assert relative(out, want.detach()) <= 4 * 3 * half
    bound = 4 * (4 * half + (2 * 2.0**-4 / 3**0.5 if ckpt else 0.0))
    for t, t64 in ((x, x64), (w1, a64), (w2, b64)):
        assert t.grad.dtype == dtype and relative(t.grad, t64.grad) <= bound
    assert (x.grad[sum(splits):] == 0).all() and (out[sum(splits):] == 0).all()
    # the calls that it is made of, one by one: the same bits
    hidden_rows = flux_amd.moe_linear(x.detach(), w1.detach(), counts(splits))
    if ckpt:
        act, codes, scale = flux_amd.moe_swiglu_checkpoint(hidden_rows)
        kept_x = flux_amd.moe_checkpoint(x.detach())
    else:
        act, codes, scale, kept_x = flux_amd.moe_swiglu(hidden_rows), hidden_rows, None, (x.detach(), None)
    assert torch.equal(out, flux_amd.moe_linear(act, w2.detach(), counts(splits)))
    grad_hidden, again = flux_amd.moe_swiglu_backward(flux_amd.moe_dgrad(up, w2.detach(), counts(splits)), codes, scale)
    assert torch.equal(w2.grad, flux_amd.moe_wgrad(up, again, counts(splits)))
    assert torch.equal(w1.grad, flux_amd.moe_wgrad(grad_hidden, kept_x[0], counts(splits), kept_x[1]))
    assert torch.equal(x.grad, flux_amd.moe_dgrad(grad_hidden, w1.detach(), counts(splits)))


def test_mlp_gradient_against_differences():
    """Along one direction: central differences of the 64-bit layer are off by h^2 of a third derivative; the gradients by their roundings (bf16, eight of them in a row)."""
    splits = [60, 40]
    x, w1, w2 = mlp_operands(splits, 0, 64, 48, BF16, 3)
    out = flux_amd.moe_mlp(x, w1, w2, counts(splits))
    up = data(out.shape, BF16, 4)
    out.backward(up)
    d = [data(t.shape, F32, 20 + i, s) for i, (t, s) in enumerate(((x, 1.0), (w1, 0.1), (w2, 0.1)))]
    at = lambda h: (mlp64(*(t.detach().double() + h * v.double() for t, v in zip((x, w1, w2), d)), splits) * up.double()).sum()  # noqa: E731
    slope = (at(1e-4) - at(-1e-4)) / 2e-4
    along = sum((t.grad.double() * v.double()).sum() for t, v in zip((x, w1, w2), d))
    spread = sum((t.grad.double() * v.double()).square().sum() for t, v in zip((x, w1, w2), d)).sqrt()  # of a sum of terms with signs at random
    assert (slope - along).abs() <= 8 * 2.0**-8 * spread * 4


@pytest.mark.parametrize("ckpt", [False, True])
def test_linear_and_swiglu_gradients(ckpt):
    splits = [33, 0, 90]
    x, w = data((130, 72), BF16, 1).requires_grad_(), data((3, 64, 72), BF16, 2).requires_grad_()
    out = flux_amd.moe_linear(x, w, counts(splits), ckpt)
    for e, r in ranges(splits, 130):
        close(out[r], x[r].detach().double() @ w[e].detach().double().t(), 72 * 2.0**-23 * (x[r].detach().double().abs() @ w[e].detach().double().abs().t()))
    assert (out[123:] == 0).all()
    gated = flux_amd.moe_swiglu(out, ckpt)
    gated.sum().backward()  # the gradient of a sum is one value with strides of 0
    ones = torch.ones_like(gated)
    kept = flux_amd.moe_swiglu_checkpoint(out.detach())[1:] if ckpt else (out.detach(), None)
    grad_out = flux_amd.moe_swiglu_backward(ones, *kept)[0]
    kept_x = flux_amd.moe_checkpoint(x.detach()) if ckpt else (x.detach(), None)
    assert torch.equal(x.grad, flux_amd.moe_dgrad(grad_out, w.detach(), counts(splits)))
    assert torch.equal(w.grad, flux_amd.moe_wgrad(grad_out, kept_x[0], counts(splits), kept_x[1]))


def test_gradients_that_are_not_wanted():
    splits = [20, 11]
    up = data((31, 64), BF16, 9)
    whole = mlp_operands(splits, 0, 64, 32, BF16)
    flux_amd.moe_mlp(*whole, counts(splits)).backward(up)
    for wanted in range(1, 7):
        leaves = [t.detach().requires_grad_(bool(wanted >> i & 1)) for i, t in enumerate(whole)]
        flux_amd.moe_mlp(*leaves, counts(splits)).backward(up)
        for t, full in zip(leaves, whole):
            assert (t.grad is None) if not t.requires_grad else torch.equal(t.grad, full.grad)
    x, w = whole[0].detach(), whole[1].detach()
    for xr, wr in ((True, False), (False, True)):
        a, b = x.clone().requires_grad_(xr), w.clone().requires_grad_(wr)
        flux_amd.moe_linear(a, b, counts(splits)).sum().backward()
        assert (a.grad is not None) == xr and (b.grad is not None) == wr


def test_kept_memory_is_halved():
    """What a layer keeps for its backward pass, without the weights."""
    splits = [2048, 2048]
    x, w1, w2 = (t.detach() for t in mlp_operands(splits, 0, 512, 1024, BF16))
    kept = {}
    for ckpt in (False, True):
        leaf = [t.clone().requires_grad_() for t in (x, w1, w2)]
        torch.cuda.synchronize()
        inputs = torch.cuda.memory_allocated()
        y = flux_amd.moe_mlp(*((leaf[0] * 1), leaf[1], leaf[2]), counts(splits), checkpoint=ckpt)
        kept[ckpt] = torch.cuda.memory_allocated() - inputs - y.numel() * 2
        del y
    assert kept[True] <= kept[False] * (33 / 64) + (1 << 16)


def layer(x, idx, weights, splits, w1, w2, ckpt):
    rows = flux_amd.moe_permute(x, idx)
    return flux_amd.moe_unpermute(flux_amd.moe_mlp(rows, w1, w2, splits, checkpoint=ckpt), idx, weights)


@pytest.mark.parametrize("ckpt", [False, True])
def test_a_whole_layer(ckpt):
    """Routing, rows to their experts, the experts, and back: dropped pairs have no row, and rows behind the last one no expert."""
    tokens, topk, experts, hidden, ffn = 200, 2, 8, 128, 64
    choosed = torch.randint(0, experts + 1, (tokens, topk), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(DEV)  # `experts`: dropped
    splits, _, idx, _, _ = capi.route_sort(choosed, experts)
    weights = torch.rand(tokens, topk, generator=torch.Generator().manual_seed(2)).to(DEV).requires_grad_()
    x = data((tokens, hidden), BF16, 3).requires_grad_()
    w1, w2 = (data(s, BF16, 4 + i, 0.1).requires_grad_() for i, s in enumerate(((experts, 2 * ffn, hidden), (experts, hidden, ffn))))
    up = data((tokens, hidden), BF16, 8)
    layer(x, idx, weights, splits, w1, w2, ckpt).backward(up)
    x64, p64, a64, b64 = (t.detach().double().requires_grad_() for t in (x, weights, w1, w2))
    out = torch.zeros(tokens, hidden, dtype=torch.float64, device=DEV)
    for e in range(experts):
        for j in range(topk):
            t = (choosed[:, j] == e).nonzero().flatten()
            h = x64[t] @ a64[e].t()
            out = out.index_add(0, t, p64[t, j, None] * ((torch.nn.functional.silu(h[:, :ffn]) * h[:, ffn:]) @ b64[e].t()))
    out.backward(up.double())
    bound = 4 * (6 * 2.0**-8 + (2 * 2.0**-4 / 3**0.5 if ckpt else 0.0))
    for t, t64 in ((x, x64), (weights, p64), (w1, a64), (w2, b64)):
        assert relative(t.grad, t64.grad) <= bound


def test_second_derivatives_are_refused():
    splits = [20, 11]
    x, w1, w2 = mlp_operands(splits, 0, 64, 32, BF16)
    for out in (flux_amd.moe_mlp(x, w1, w2, counts(splits)), flux_amd.moe_linear(x, w1, counts(splits)), flux_amd.moe_swiglu(x)):
        with pytest.raises(RuntimeError, match="gradient of the gradient"):
            torch.autograd.grad(out.sum(), [x], create_graph=True)


# ---- streams, graphs, refusals -------------------------------------------------------------------------------------


def test_on_another_stream():
    splits = counts([300, 212])
    x, w1, w2 = (t.detach() for t in mlp_operands([300, 212], 0, 256, 128, BF16))
    want = flux_amd.moe_wgrad(x * 2, x, splits), flux_amd.moe_dgrad(flux_amd.moe_linear(x * 2, w1, splits), w1, splits)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = x * 2
        got = flux_amd.moe_wgrad(y, x, splits), flux_amd.moe_dgrad(flux_amd.moe_linear(y, w1, splits), w1, splits)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once():
    """Workspaces are each call's own: weights' gradients in parts, on two streams at the same time."""
    splits = counts([5000, 3000])
    a, b = [data((8000, 128), BF16, i) for i in (1, 2)], [data((8000, 128), BF16, i) for i in (3, 4)]
    assert capi.load().fluxmi_moe_wgrad_workspace_bytes(2, 8000, 128, 128) > 0
    want = [flux_amd.moe_wgrad(*p, splits) for p in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for s, p in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(flux_amd.moe_wgrad(*p, splits))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))


# Weights' gradients whose tiles are fetched from queues, and both gradients with tiles that are cut: (rows, experts, n, k)
WORKSPACES = [("wgrad", 2600, 64, 1024, 1024), ("wgrad", 5001, 2, 1544, 1288), ("dgrad", 90, 3, 4104, 264), ("dgrad", 700, 2, 4096, 520)]


def workspace_call(kind, rows, experts, n, k, seed):
    grad, other = data((rows, n), BF16, seed), data((rows, k) if kind == "wgrad" else (experts, n, k), BF16, seed + 1)
    size = getattr(capi.load(), f"fluxmi_moe_{kind}_workspace_bytes")(experts, rows, n, k)
    assert size > 0
    call = flux_amd.moe_wgrad if kind == "wgrad" else flux_amd.moe_dgrad
    return grad, lambda splits: call(grad, other, splits)


def some_counts(rows, experts, seed):
    g = torch.Generator().manual_seed(seed)
    cuts = torch.randint(0, rows + 1, (experts,), generator=g).sort().values
    return counts(torch.diff(cuts, prepend=torch.tensor([0])).tolist())


@pytest.mark.parametrize("kind,rows,experts,n,k", WORKSPACES)
def test_workspaces_on_two_streams_at_once(kind, rows, experts, n, k):
    splits = some_counts(rows, experts, 1)
    both = [workspace_call(kind, rows, experts, n, k, seed) for seed in (1, 3)]
    want = [call(splits) for _, call in both]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(6):
        for s, (_, call) in zip(streams, both):
            with torch.cuda.stream(s):
                got.append(call(splits))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))


@pytest.mark.parametrize("kind,rows,experts,n,k", WORKSPACES)
def test_workspaces_in_two_graphs(kind, rows, experts, n, k):
    """Two graphs out of one pool of memory, replayed in turn, with other operands and row counts and eager work between."""
    splits = some_counts(rows, experts, 1)
    both = [workspace_call(kind, rows, experts, n, k, seed) for seed in (1, 3)]
    for _, call in both:
        call(splits)
    torch.cuda.synchronize()
    graphs, pool = [], torch.cuda.graph_pool_handle()
    for _, call in both:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            got = call(splits)
        graphs.append((g, got))
    for seed in (1, 5, 7):
        splits.copy_(some_counts(rows, experts, seed))
        for (grad, call), (g, got) in zip(both, graphs):
            grad.copy_(data(grad.shape, BF16, 20 + seed))
            want = call(splits)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


@pytest.mark.parametrize("pinned", [False, True])
def test_graph_with_row_counts_on_the_host(pinned):
    """A replay reads the counts again from the tensor that the captured call was given."""
    x, w = data((40, 64), BF16, 1), data((4, 72, 64), BF16, 2)
    splits = torch.tensor([10, 0, 25, 5], dtype=torch.int32)
    splits = splits.pin_memory() if pinned else splits

    def run(splits):
        y = flux_amd.moe_linear(x, w, splits)
        return y, flux_amd.moe_dgrad(y, w, splits), flux_amd.moe_wgrad(y, x, splits)

    run(splits)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run(splits)
    for new in ([10, 0, 25, 5], [1, 2, 3, 4], [40, 0, 0, 0], [0, 0, 0, 0]):
        want = run(counts(new))
        splits.copy_(torch.tensor(new, dtype=torch.int32))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("ckpt", [False, True])
def test_graph_of_a_training_step_replays(ckpt):
    """Forward and backward in two graphs, with eager work between the replays and other row counts each time; weights' gradients in parts among it."""
    rows, hidden, ffn = 3000, 64, 48
    splits = counts([1000, 0, 1900])
    x, w1, w2 = (t.detach() for t in mlp_operands([1000, 0, 1900], 100, hidden, ffn, BF16))
    up = data((rows, hidden), BF16, 7)
    assert capi.load().fluxmi_moe_wgrad_workspace_bytes(3, rows, hidden, ffn) > 0

    def step():
        h = flux_amd.moe_linear(x, w1, splits)
        if ckpt:
            act, kept, scale = flux_amd.moe_swiglu_checkpoint(h)
            kept_x = flux_amd.moe_checkpoint(x)
        else:
            act, kept, scale, kept_x = flux_amd.moe_swiglu(h), h, None, (x, None)
        out = flux_amd.moe_linear(act, w2, splits)
        grad_h, act = flux_amd.moe_swiglu_backward(flux_amd.moe_dgrad(up, w2, splits), kept, scale)
        return out, flux_amd.moe_wgrad(up, act, splits), flux_amd.moe_wgrad(grad_h, kept_x[0], splits, kept_x[1], output_dtype=F32), flux_amd.moe_dgrad(grad_h, w1, splits)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step()
        graphs.append((g, got))
    for seed, new in enumerate(([1000, 0, 1900], [0, 3000, 0], [7, 8, 9], [0, 0, 0])):
        x.copy_(data(x.shape, BF16, 20 + seed))
        splits.copy_(counts(new))
        want = step()
        for g, got in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_backward_pass():
    """The recorded gradients in a graph; refused while an eager graph of the same leaves is alive, whose stream the capture would draw in."""
    splits = counts([30, 33])
    x, w1, w2 = mlp_operands([30, 33], 1, 64, 32, BF16)
    for make in (lambda: flux_amd.moe_mlp(x, w1, w2, splits), lambda: flux_amd.moe_linear(x, w1, splits), lambda: flux_amd.moe_swiglu(x)):
        alive = flux_amd.moe_mlp(x, w1, w2, splits)
        g = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
            with torch.cuda.graph(g):
                make().sum().backward()
        del alive, g
        x.grad = w1.grad = w2.grad = None

    def step():
        return torch.autograd.grad(flux_amd.moe_mlp(x, w1, w2, splits, checkpoint=True).float().square().mean(), [x, w1, w2])

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for seed in range(3):
        with torch.no_grad():
            x.copy_(data(x.shape, BF16, 40 + seed))
        want = step()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    x, w, splits = data((10, 64), BF16, 1), data((2, 32, 64), BF16, 2), counts([4, 6])
    codes, scale = flux_amd.moe_checkpoint(x)
    both = torch.zeros(200, 64, dtype=BF16, device=DEV)
    bad = [
        (lambda: flux_amd.moe_linear(x.float(), w, splits), "bfloat16 or float16"),
        (lambda: flux_amd.moe_linear(x, w.half(), splits), "weight is Half"),
        (lambda: flux_amd.moe_linear(x[:, :32].contiguous(), w, splits), "mismatch"),
        (lambda: flux_amd.moe_linear(x[:, ::2], w, splits), "contiguous"),
        (lambda: flux_amd.moe_linear(x, w, splits.long()), "int32"),
        (lambda: flux_amd.moe_linear(x, w, counts([10])), "splits 0-dim mismatch"),
        (lambda: flux_amd.moe_linear(x, w, counts([4, 0, 6, 0])[::2]), "contiguous"),
        (lambda: flux_amd.moe_dgrad(x, w, splits), "mismatch"),
        (lambda: flux_amd.moe_wgrad(x, x[:9], splits), "rows"),
        (lambda: flux_amd.moe_wgrad(x, codes, splits), "bfloat16 or float16"),
        (lambda: flux_amd.moe_wgrad(x, x, splits, scale), "float8_e4m3fn"),
        (lambda: flux_amd.moe_wgrad(x, codes, splits, scale[:, :1]), "contiguous"),
        (lambda: flux_amd.moe_wgrad(x, codes, splits, scale[:9]), "shape mismatch"),
        (lambda: flux_amd.moe_wgrad(x, x, splits, output_dtype=F16), "float32"),
        (lambda: flux_amd.moe_wgrad(x, x, splits, accumulate=True), "accumulate needs an output"),
        (lambda: flux_amd.moe_wgrad(x, x, splits, output=torch.zeros(2, 64, 63, device=DEV)), "shape mismatch"),
        (lambda: flux_amd.moe_wgrad(x, x, splits, output=torch.zeros(2, 64, 64, device=DEV), output_dtype=BF16), "output is"),
        (lambda: flux_amd.moe_wgrad(x, x, splits, output=torch.zeros(2, 64, 64, device=DEV, requires_grad=True)), "no_grad"),
        (lambda: flux_amd.moe_wgrad(x, x, splits, output=torch.zeros(2 * 64 * 64 + 1, device=DEV)[1:].view(2, 64, 64)), "aligned"),
        (lambda: flux_amd.moe_wgrad(both[:10], x, splits, output=both[9:].view(-1)[:2 * 64 * 64].view(2, 64, 64)), "memory of an operand"),
        (lambda: flux_amd.moe_wgrad(x, codes, splits, scale, output=torch.zeros(2, 64, 64, device=DEV)._neg_view()), "negative view"),
        (lambda: flux_amd.moe_swiglu(x[:, :63].contiguous()), "gate and up"),
        (lambda: flux_amd.moe_swiglu_backward(x, x), "shape mismatch"),
        (lambda: flux_amd.moe_swiglu_backward(x[:, :32].contiguous(), codes, scale[:, :1].contiguous()), "shape mismatch"),
        (lambda: flux_amd.moe_mlp(x, w, data((2, 64, 15), BF16, 3), splits), "gate and up"),
        (lambda: flux_amd.moe_mlp(x, w, data((3, 64, 16), BF16, 3), splits), "experts"),
        (lambda: flux_amd.moe_checkpoint(x.view(-1)), "2 dimensions"),
        (lambda: flux_amd.moe_linear(x, torch.zeros(1025, 8, 64, dtype=BF16, device=DEV), counts([0] * 1025)), "1024 experts"),
        (lambda: flux_amd.moe_linear(torch.empty((1 << 24) + 1, 8, dtype=BF16, device=DEV), torch.zeros(1, 8, 8, dtype=BF16, device=DEV), counts([1])), "2\\^24 rows"),
    ]
    for call, text in bad:
        with pytest.raises(RuntimeError, match=text):
            call()


def test_empty_sizes():
    splits = counts([0, 0])
    x, w = data((0, 64), BF16, 1), data((2, 32, 64), BF16, 2)
    assert flux_amd.moe_linear(x, w, splits).shape == (0, 32) and flux_amd.moe_dgrad(data((0, 32), BF16, 1), w, splits).shape == (0, 64)
    dw = flux_amd.moe_wgrad(data((0, 32), BF16, 1), x, splits)
    assert dw.shape == (2, 32, 64) and not dw.any()
    for kept in (None, torch.empty(0, 33, dtype=torch.float8_e8m0fnu, device=DEV)):  # the same by tiles
        dw = flux_amd.moe_wgrad(data((0, 1032), BF16, 1), data((0, 1040), BF16, 1) if kept is None else torch.empty(0, 1040, dtype=torch.float8_e4m3fn, device=DEV), counts([0] * 8), kept)
        assert dw.shape == (8, 1032, 1040) and not dw.any()
    assert not flux_amd.moe_dgrad(data((300, 2056), BF16, 1), data((2, 2056, 64), BF16, 2), splits).any()
    assert flux_amd.moe_checkpoint(x)[1].shape == (0, 2) and flux_amd.moe_swiglu(x).shape == (0, 32)
    x, w1, w2 = mlp_operands([0, 0], 0, 64, 32, BF16)
    flux_amd.moe_mlp(x, w1, w2, splits).sum().backward()
    assert x.grad.shape == (0, 64) and not w1.grad.any() and not w2.grad.any()
