"""MXFP4 on the GPU: quantisation bit for bit against the oracle, products against 64 bits.

A product's bound: the terms are exact in fp32 (two 2-bit significands and powers of two), their sum in fp32 is off by at most K roundings of 2^-24 of the
sum of magnitudes, and the result is rounded to its type once (half a step, eps / 2), after one more rounding by row_scale."""
import numpy as np
import pytest
import torch

import flux_amd
from flux_amd import capi
from oracle import mx

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
FP4, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


def quantiser(dtype):
    return flux_amd.Quantization(dtype, FP4)


def bytes_of(t):
    return t.view(torch.uint8).cpu().numpy()


def hard_values(rows, cols, dtype, seed):
    """Blocks of every magnitude the type has, ties, zeros of both signs, subnormal values, and a few blocks with an infinity or a NaN."""
    rng = np.random.default_rng(seed)
    info = torch.finfo(dtype)
    lo, hi = np.log2(info.tiny * info.eps), np.log2(info.max) - 1
    size = np.exp2(rng.uniform(lo, hi, (rows, (cols + 31) // 32))).repeat(32, axis=1)[:, :cols]
    x = rng.standard_normal((rows, cols)) * size / 4
    tie = rng.random((rows, cols)) < 0.2
    quarter = np.exp2(np.floor(np.log2(size)))
    x = np.where(tie, np.round(x / quarter * 4) / 4 * quarter, x)
    x = np.where(rng.random((rows, cols)) < 0.05, 0.0, x)
    x = np.where(rng.random((rows, cols)) < 0.02, -0.0, x)
    x = np.where(rng.random((rows, 1)) < 0.05, 0.0, x)
    bad = rng.random((rows, cols)) < 0.0005
    x = np.where(bad, rng.choice([np.inf, -np.inf, np.nan], (rows, cols)), x)
    return torch.from_numpy(x).clamp(-info.max, info.max).where(torch.from_numpy(~bad), torch.from_numpy(x)).to(dtype)


SHAPES = [(1, 32), (1, 1), (3, 31), (7, 33), (128, 7168), (50, 2048), (33, 1000), (257, 96), (300, 130), (2, 16384), (1000, 64), (515, 2056), (2100, 2050), (1030, 4112), (4100, 4160)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantise_bit_for_bit(rows, cols, dtype):
    print(f"[case] quantise {rows} {cols} {dtype}", flush=True)
    x = hard_values(rows, cols, dtype, rows + cols)
    q = quantiser(dtype)
    want = mx.quantise(x.double().numpy())
    want_t = mx.quantise(x.double().numpy().T)
    codes, scale, none, none2 = q.quantize_mx(x.to(DEV))
    assert none is None and none2 is None and codes.dtype == FP4 and scale.dtype == E8M0
    assert np.array_equal(bytes_of(scale), want[1]) and np.array_equal(bytes_of(codes), want[0])
    codes, scale, codes_t, scale_t = q.quantize_mx(x.to(DEV), return_tranpose=True)
    assert np.array_equal(bytes_of(scale), want[1]) and np.array_equal(bytes_of(codes), want[0])
    assert np.array_equal(bytes_of(scale_t), want_t[1]) and np.array_equal(bytes_of(codes_t), want_t[0])
    # and back: the values are held by the type
    for c, s, n, (wc, ws) in ((codes, scale, cols, want), (codes_t, scale_t, rows, want_t)):
        back = q.dequantize_mx(c, s, n)
        assert back.dtype == dtype and np.array_equal(back.double().cpu().numpy(), mx.values(wc, ws)[:, :n], equal_nan=True)


def test_large_and_flat_forms():
    """Enough values for the form with four groups in flight, and a tensor whose last workgroup is not full."""
    for rows, cols, dtype in ((4099, 1056, BF16), (2051, 4096, F32), (4100, 1056, F16)):
        x = (torch.randn(rows, cols, generator=torch.Generator().manual_seed(1)) * 3).to(dtype)
        codes, scale, _, _ = quantiser(dtype).quantize_mx(x.to(DEV))
        want = mx.quantise(x.double().numpy())
        assert np.array_equal(bytes_of(scale), want[1]) and np.array_equal(bytes_of(codes), want[0])
        back = quantiser(dtype).dequantize_mx(codes, scale)
        assert np.array_equal(back.double().cpu().numpy(), mx.values(*want))


@pytest.mark.parametrize("cols", [2080, 2051])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_values_of_many_megabytes_as_their_parts(dtype, cols):
    """From 96 MB on the values pass the caches by; parts of 32 x 100 rows are below that."""
    rows = (112 << 20) // (cols * (4 if dtype == F32 else 2))
    x = torch.randn(rows, cols, device=DEV, generator=torch.Generator(DEV).manual_seed(cols)).mul_(5).to(dtype)
    q = quantiser(dtype)
    codes, scale, codes_t, scale_t = (t.view(torch.uint8) for t in q.quantize_mx(x, True))
    along = [t.view(torch.uint8) for t in q.quantize_mx(x)[:2]]
    assert torch.equal(codes, along[0]) and torch.equal(scale, along[1])
    back = q.dequantize_mx(codes.view(FP4), scale.view(E8M0), cols)
    for lo in range(0, rows, 3200):
        part, blocks = x[lo:lo + 3200], slice(lo // 32, lo // 32 + 100)
        c, s, ct, st = (t.view(torch.uint8) for t in q.quantize_mx(part, True))
        assert torch.equal(codes[lo:lo + 3200], c) and torch.equal(scale[lo:lo + 3200], s)
        assert torch.equal(codes_t[:, lo // 2:lo // 2 + 1600], ct) and torch.equal(scale_t[:, blocks], st)
        assert torch.equal(back[lo:lo + 3200], q.dequantize_mx(c.view(FP4), s.view(E8M0), cols))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_batch_of_matrices(dtype):
    x = hard_values(5 * 70, 100, dtype, 4).view(5, 70, 100)
    for transposed in (False, True):
        codes, scale, codes_t, scale_t = quantiser(dtype).quantize_mx(x.to(DEV), transposed)
        want = mx.quantise(x.double().numpy())
        assert codes.shape == (5, 70, 64) and np.array_equal(bytes_of(codes), want[0]) and np.array_equal(bytes_of(scale), want[1])
        if transposed:
            want = mx.quantise(x.double().numpy().transpose(0, 2, 1))
            assert codes_t.shape == (5, 100, 48) and np.array_equal(bytes_of(codes_t), want[0]) and np.array_equal(bytes_of(scale_t), want[1])


def test_batch_of_large_matrices():
    x = torch.randn(3, 1211, 1250, device=DEV, generator=torch.Generator(DEV).manual_seed(1)).to(BF16)
    whole = quantiser(BF16).quantize_mx(x, True)
    for i in range(3):
        for a, b in zip(whole, quantiser(BF16).quantize_mx(x[i], True)):
            assert torch.equal(a[i].view(torch.uint8), b.view(torch.uint8))


def test_dequantise_every_code_and_scale():
    codes = torch.arange(256, dtype=torch.uint8).repeat_interleave(16).view(1, -1).repeat(256, 1)     # every byte in a block of its own
    scale = torch.arange(256, dtype=torch.uint8).view(256, 1).repeat(1, 256)
    want = mx.values(codes.numpy(), scale.numpy())
    for dtype in (F32, BF16, F16):
        got = quantiser(dtype).dequantize_mx(codes.to(DEV).view(FP4), scale.to(DEV).view(E8M0))
        expect = torch.from_numpy(want).to(F32).to(dtype)  # (fp32 holds them all but 6 * 2^127 and 4 * 2^127, infinite there and here)
        assert torch.equal(got.cpu().nan_to_num(nan=7.0), expect.nan_to_num(nan=7.0))
        assert torch.equal(got.cpu().isnan(), expect.isnan())


def test_values_at_any_element():
    flat = hard_values(1, 3 + 40 * 70, BF16, 3).view(-1).to(DEV)
    x = flat[3:].view(40, 70)
    for t in (False, True):
        for a, b in zip(quantiser(BF16).quantize_mx(x, t), quantiser(BF16).quantize_mx(x.clone(), t)):
            assert (a is None and b is None) or np.array_equal(bytes_of(a), bytes_of(b))
    even = flat[3:3 + 2 * 1024].view(2, 1024)
    assert np.array_equal(bytes_of(quantiser(BF16).quantize_mx(even)[0]), bytes_of(quantiser(BF16).quantize_mx(even.clone())[0]))


def test_nothing_to_quantise():
    for shape in ((0, 64), (4, 0), (0, 3, 5)):
        codes, scale, codes_t, scale_t = quantiser(F32).quantize_mx(torch.empty(shape, device=DEV), True)
        assert codes.numel() == 0 and scale.numel() == 0 and codes_t.numel() == 0
    assert quantiser(F32).dequantize_mx(torch.empty(0, 16, dtype=torch.uint8, device=DEV).view(FP4),
                                        torch.empty(0, 1, dtype=torch.uint8, device=DEV).view(E8M0)).shape == (0, 32)


# ---- products ----------------------------------------------------------------------------------------------------


def operand(*shape, k, seed):
    """Codes and scales of a tensor [*shape, k]: every code, scales over a few powers of two; and its values, fp64 on the GPU."""
    g = torch.Generator().manual_seed(seed)
    kb = mx.blocks(k)
    codes = torch.randint(0, 256, (*shape, kb, 16), dtype=torch.uint8, generator=g)
    last = k - 32 * (kb - 1)  # the end of the last block is zero codes
    codes[..., -1, (last + 1) // 2:] = 0
    if last % 2:
        codes[..., -1, last // 2] &= 15
    scale = torch.randint(122, 130, (*shape, kb), dtype=torch.uint8, generator=g)
    codes = codes.view(*shape, kb * 16)
    table = torch.from_numpy(mx.values(np.arange(256, dtype=np.uint8)[:, None].repeat(16, 1), np.full((256, 1), 127, np.uint8)))[:, :2].to(DEV)
    codes, scale = codes.to(DEV), scale.to(DEV)
    # (in parts: one lookup of 2^26 codes and more is past what the library's kernel launches, and what it left out would be zeros)
    value = torch.cat([table[part.long()] for part in codes.flatten().split(1 << 22)]).view(*codes.shape[:-1], 2 * codes.shape[-1]) * torch.exp2(scale.double() - 127).repeat_interleave(32, -1)
    return codes.view(FP4), scale.view(E8M0), value


def check(got, a, w, k, factor=None):
    """got against a [M, K] @ w [N, K]^T in fp64."""
    want, size = a @ w.t(), a.abs() @ w.abs().t()
    if factor is not None:
        want, size = want * factor.double()[:, None], size * factor.double().abs()[:, None]
    step = torch.finfo(got.dtype).eps / 2 if got.dtype != F32 else 0.0
    bound = step * want.abs() + (k + 2) * 2.0**-24 * size
    off = (got.double() - want).abs()
    assert (off <= bound * 1.0000001).all(), f"off by {(off - bound).max().item():.3g} more than the bound"


@pytest.mark.parametrize("out", [BF16, F16, F32])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 64, 32), (16, 16, 128), (17, 65, 544), (5, 1000, 100), (64, 64, 512), (65, 257, 2048), (300, 130, 1056),
                                   (128, 128, 4096), (513, 520, 640), (1025, 384, 160), (2, 4096, 14336), (700, 1025, 3000)])
def test_dense_product(m, n, k, out):
    print(f"[case] dense {m} {n} {k} {out}", flush=True)
    a, sa, va = operand(m, k=k, seed=1)
    w, sw, vw = operand(n, k=k, seed=2)
    got = flux_amd.MxGemm(out).forward(a, w, sa, sw)
    assert got.shape == (m, n) and got.dtype == out
    check(got, va, vw, k)


SPLITS = [[0, 3, 0, 70], [5], [1, 1, 1, 1, 1], [0, 0, 0], [200, 0, 16, 33], [64, 64, 128], [129, 1, 255, 31, 0, 300], [600, 2, 0, 900], [17] * 70]


@pytest.mark.parametrize("n,k", [(96, 224), (257, 1100), (512, 2048)])
@pytest.mark.parametrize("splits", SPLITS, ids=str)
@pytest.mark.parametrize("gathered,weighted,out", [(False, False, BF16), (True, False, F16), (False, True, F32), (True, True, BF16)])
def test_grouped_product(splits, n, k, gathered, weighted, out):
    print(f"[case] grouped {splits} {n} {k} {gathered} {weighted} {out}", flush=True)
    rows, experts = sum(splits), len(splits)
    tokens = max(rows // 3, 1) if gathered else rows
    a, sa, va = operand(tokens, k=k, seed=3)
    w, sw, vw = operand(experts, n, k=k, seed=4)
    extra = 9  # rows past the last routed one are left as they were
    g = torch.Generator().manual_seed(5)
    gather = torch.randint(0, tokens, (rows + extra,), generator=g).to(torch.int32).to(DEV) if gathered else None
    if not gathered:
        a, sa = (torch.cat([t.view(torch.uint8), t.view(torch.uint8).new_full((extra, t.shape[1]), 255)]).view(t.dtype) for t in (a, sa))
    factor = torch.rand(rows + extra, generator=g).to(DEV) if weighted else None
    sp = torch.tensor(splits, dtype=torch.int32)
    got = torch.full((rows + extra, n), 77.0, dtype=out, device=DEV)
    same = flux_amd.MxGemm(out).forward_grouped(a, sp.to(DEV), w, sa, sw, gather_index=gather, row_scale=factor, output=got)
    assert same.data_ptr() == got.data_ptr() and (got[rows:] == 77).all()
    at = 0
    for e, r in enumerate(splits):
        mine = slice(at, at + r)
        check(got[mine], va[gather[mine].long()] if gathered else va[mine], vw[e], k, factor[mine] if weighted else None)
        at += r
    host = flux_amd.MxGemm(out).forward_grouped(a, sp, w, sa, sw, gather_index=gather, row_scale=factor)
    assert torch.equal(host[:rows], got[:rows])


def grouped(splits, n, k, out, seed=3):
    """A grouped product of random operands, checked expert by expert."""
    rows = sum(splits)
    a, sa, va = operand(rows, k=k, seed=seed)
    w, sw, vw = operand(len(splits), n, k=k, seed=seed + 1)
    factor = torch.rand(rows, generator=torch.Generator().manual_seed(seed)).to(DEV)
    got = flux_amd.MxGemm(out).forward_grouped(a, torch.tensor(splits, dtype=torch.int32, device=DEV), w, sa, sw, row_scale=factor)
    at = 0
    for e, r in enumerate(splits):
        check(got[at:at + r], va[at:at + r], vw[e], k, factor[at:at + r])
        at += r


def brief(v):
    return f"{sum(v)}of{len(v)}" if isinstance(v, list) else str(v)


# Streams of 16 and of 32 rows whose waves split K in four, in two and not at all, by the number of pieces (experts with rows times n / 32).
@pytest.mark.parametrize("k", [512, 1024, 2560, 8192])
@pytest.mark.parametrize("splits,n", [([1, 1], 500), ([3] * 8, 1000), ([9, 1] * 16, 1000), ([30, 17], 500), ([16, 20, 1, 33, 0, 15, 17, 28], 1000),
                                      ([13, 0] * 15 + [40, 60], 800), ([20, 12] * 16, 1030)], ids=brief)
def test_streams(splits, n, k):
    for out in (BF16, F32):
        print(f"[case] streams {splits} {n} {k} {out}", flush=True)
        grouped(splits, n, k, out)


# Panels of 64 rows (experts with rows times n / 128 is 240 or more, 48 rows on average at most) and of 128: rows that end in each block of 16 and past the panel's.
@pytest.mark.parametrize("k", [512, 1024, 2560, 7168])
@pytest.mark.parametrize("splits,n", [([1, 0, 2] * 20, 900), ([16, 17, 31, 32, 33, 63, 64, 65, 0, 2] * 4, 1000), ([150, 1, 1, 1, 129, 2, 3, 70] * 4, 1030),
                                      ([100, 127, 128, 129, 16, 200, 17, 90] * 2, 2000), ([97, 33, 128, 1, 130] * 8, 1001), ([700], 3001)], ids=brief)
def test_panels(splits, n, k):
    for out in (BF16, F16, F32):
        print(f"[case] panels {splits} {n} {k} {out}", flush=True)
        grouped(splits, n, k, out)


@pytest.mark.parametrize("k", [32, 384, 1408, 2816, 2880, 705])
@pytest.mark.parametrize("splits,n", [([1, 1], 500), ([30, 17], 500), ([3] * 20, 1600), ([16, 31, 33, 64, 65, 0] * 5, 1100), ([100, 129, 60, 200] * 4, 2001), ([700, 20], 512),
                                      ([256, 150, 257, 16, 200, 180, 255, 129] * 2, 1601), ([600, 0, 33, 256, 257], 5000), ([3000], 1301), ([70, 52] * 65, 300)], ids=brief)
def test_rows_that_end_inside_a_line(splits, n, k):
    """Every form with K that is a multiple of 128 (scales on whole words) and not."""
    for out in (BF16, F32):
        print(f"[case] ends {splits} {n} {k} {out}", flush=True)
        grouped(splits, n, k, out)


@pytest.mark.parametrize("k", [544, 640, 1056, 1408, 2880, 4128])
@pytest.mark.parametrize("splits,n", [([300, 0, 257, 700, 65], 5000), ([512] * 3, 8192), ([64, 200, 1, 129] * 8, 4104)], ids=brief)
def test_tiles_of_rows_that_end_inside_a_line(splits, n, k):
    for out in (BF16, F16, F32):
        print(f"[case] tiles, ends {splits} {n} {k} {out}", flush=True)
        grouped(splits, n, k, out)


@pytest.mark.parametrize("experts,rows,n", [(4, 300, 5000), (2, 3, 300), (2, 20, 300), (12, 9, 2600), (16, 100, 2000), (3, 600, 520), (16, 200, 1601)])
@pytest.mark.parametrize("k", [384, 640, 736, 1152])
def test_nan_blocks_beside_the_ends_of_rows(experts, rows, n, k):
    """What lies behind a row's last scale is the next row's first: a NaN block there stays there."""
    a, sa, va = operand(experts * rows, k=k, seed=1)
    w, sw, vw = operand(experts, n, k=k, seed=2)
    sa.view(torch.uint8)[1::2, 0] = 255
    sw.view(torch.uint8)[:, 1::2, 0] = 255
    got = flux_amd.MxGemm(F32).forward_grouped(a, torch.full((experts,), rows, dtype=torch.int32, device=DEV), w, sa, sw)
    row, col = torch.arange(experts * rows, device=DEV) % 2 == 1, torch.arange(n, device=DEV) % 2 == 1
    assert torch.equal(got.isnan(), row[:, None] | col[None])
    for e in range(experts):
        mine = torch.arange(e * rows, (e + 1) * rows, device=DEV)
        mine = mine[mine % 2 == 0]
        check(got[mine][:, ::2], va[mine], vw[e][::2], k)


# Tiles of 256 x 256: rows that end in each of a tile's four units of 64, experts without rows, columns that end in each half and quarter of a tile; as many as an
# expert table holds and one more; results whose rows are and are not whole stores.
@pytest.mark.parametrize("out", [BF16, F16, F32])
@pytest.mark.parametrize("splits,n,k", [([300, 0, 1, 700], 520, 1024), ([64, 65, 128, 129, 192, 193, 256, 257], 264, 1536), ([1000, 31], 72, 2048),
                                        ([513], 1160, 512), ([511], 136, 4096), ([2000, 1], 2048, 1024), ([40] * 128, 64, 1024), ([30] * 129, 64, 1024),
                                        ([200, 300], 516, 1024), ([200, 300], 514, 1024), ([26] * 32, 2048, 1024), ([20] * 32, 2048, 1024)], ids=brief)
def test_tiles(splits, n, k, out):
    print(f"[case] tiles {splits} {n} {k} {out}", flush=True)
    grouped(splits, n, k, out)


@pytest.mark.parametrize("rows", [5, 100, 700])
def test_operands_that_are_parts_of_others(rows):
    """Scales from any byte on, codes from any row: blocks of a row are not a multiple of 16."""
    for k in (320, 1024):
        a, sa, va = operand(rows + 3, k=k, seed=1)
        w, sw, vw = operand(3, 130, k=k, seed=2)
        got = flux_amd.MxGemm(F32).forward(a[3:], w[1], sa[3:], sw[1])
        check(got, va[3:], vw[1], k)
        moved = sa.view(torch.uint8).new_empty(sa.numel() + 1)[1:].view(sa.shape)
        moved.copy_(sa.view(torch.uint8))
        assert torch.equal(flux_amd.MxGemm(F32).forward(a[3:], w[1], moved[3:].view(E8M0), sw[1]), flux_amd.MxGemm(F32).forward(a[3:], w[1].clone(), moved[3:].view(E8M0), sw[1].clone()))
        check(flux_amd.MxGemm(F32).forward(a[3:], w[1], moved[3:].view(E8M0), sw[1]), va[3:], vw[1], k)


def test_two_streams_at_once():
    """Calls of every form, each on two streams that run together, and the same results as one after another."""
    calls = []
    for rows, n, k in ((4, 700, 2048), (40, 700, 2048), (600, 704, 2048), (600, 700, 2016), (9, 700, 2016), (600, 5000, 2048), (300, 6000, 2048)):
        a, sa, _ = operand(rows, k=k, seed=rows)
        w, sw, _ = operand(n, k=k, seed=rows + 1)
        calls.append(lambda a=a, w=w, sa=sa, sw=sw: flux_amd.MxGemm(BF16).forward(a, w, sa, sw))
    want = [call() for call in calls]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for which in (0, 1):
            with torch.cuda.stream(streams[which]):
                got[which] += [call() for call in calls]
    torch.cuda.synchronize()
    for results in got:
        for i, result in enumerate(results):
            assert torch.equal(result, want[i % len(calls)])


def test_counts_below_zero_and_past_the_rows():
    a, sa, va = operand(40, k=256, seed=1)
    w, sw, vw = operand(4, 70, k=256, seed=2)
    out = torch.full((40, 70), 5.0, device=DEV)
    flux_amd.MxGemm(F32).forward_grouped(a, torch.tensor([10, -7, 25, 1 << 30], dtype=torch.int32, device=DEV), w, sa, sw, output=out)
    for e, rows in ((0, slice(0, 10)), (2, slice(10, 35)), (3, slice(35, 40))):
        check(out[rows], va[rows], vw[e], 256)


def form_of(splits, extra, n, k, tokens=None):
    info, _ = capi.mx_launch_info(len(splits), sum(splits) + extra, n, k, a_rows=tokens)
    return info.form, info.rows, info.cols, info.waves


FEW, STREAM, PANEL, DUAL, TILES = capi.MX_FEW_ROWS, capi.MX_STREAM, capi.MX_PANEL, capi.MX_DUAL, capi.MX_TILES
# Every kernel of the products: K that ends in each part of its steps, rows of experts that end in each unit of its pieces, columns that are not whole ones; the dual
# tiles' table of two experts to a lane (66 and 100) and what keeps them off (K up to 512, 130 experts).
FORMS = [([5, 0, 3], 300, 705, (FEW, 16, 64, 4)), ([16, 0, 15, 1, 16] * 3, 1001, 2880, (FEW, 16, 64, 4)),
         ([5, 0, 3], 300, 640, (STREAM, 16, 32, 4)), ([5, 0, 3, 8] * 5, 1001, 640, (STREAM, 16, 32, 2)), ([5, 0, 3, 8] * 7, 1001, 1024, (STREAM, 16, 32, 1)),
         ([17, 30], 300, 640, (STREAM, 32, 32, 4)), ([40, 20], 300, 705, (STREAM, 32, 32, 4)), ([17, 30, 20, 40], 4000, 640, (STREAM, 32, 32, 2)),
         ([128], 4096, 384, (STREAM, 32, 32, 1)), ([17, 30, 20, 40, 60, 50], 3001, 1408, (STREAM, 32, 64, 1)),
         ([40, 17, 64, 65, 0, 33, 50, 51], 3001, 640, (PANEL, 64, 128, 1)), ([260], 4095, 705, (PANEL, 64, 128, 1)),
         ([150, 1, 250, 129, 470], 3001, 640, (PANEL, 128, 128, 1)), ([256, 300], 4000, 1056, (PANEL, 128, 128, 1)),
         ([300, 0, 257, 700, 65, 1, 512, 130], 2305, 640, (DUAL, 256, 256, 1)), ([300, 0, 257, 700, 65, 1, 512, 130], 2305, 544, (DUAL, 256, 256, 1)),
         ([64, 193, 600, 256, 0, 128, 449, 300], 2312, 1536, (DUAL, 256, 256, 1)), ([70, 52] * 50, 400, 640, (DUAL, 256, 256, 1)),
         ([70, 0, 150, 5] * 16 + [3, 200], 501, 1056, (DUAL, 256, 256, 1)),
         ([300, 0, 257, 700, 65, 1, 512, 130], 2305, 384, (TILES, 256, 256, 1)), ([300, 0, 257, 700, 65, 1, 512, 130], 2304, 512, (TILES, 256, 256, 1)),
         ([70, 52] * 65, 300, 1408, (TILES, 256, 256, 1))]


@pytest.mark.parametrize("gathered,weighted,out", [(False, True, F32), (True, False, BF16), (True, True, F16)])
@pytest.mark.parametrize("splits,n,k,form", FORMS, ids=brief)
def test_every_form(splits, n, k, form, gathered, weighted, out):
    """Rows that are gathered from fewer (entries past them are clamped), and rows past the splits' sum that stay as they were, in every kernel."""
    print(f"[case] form {form} {brief(splits)} {n} {k} {gathered} {weighted} {out}", flush=True)
    rows, extra = sum(splits), 9
    tokens = max(rows // 3, 1) if gathered else None
    assert form_of(splits, extra, n, k, tokens) == form
    g = torch.Generator().manual_seed(5)
    a, sa, va = operand(tokens or rows, k=k, seed=3)
    w, sw, vw = operand(len(splits), n, k=k, seed=4)
    gather, source = None, torch.arange(rows, device=DEV)
    if gathered:
        entries = torch.randint(0, tokens, (rows + extra,), generator=g)
        entries[1::7], entries[2::11], entries[3::13] = tokens, -5, 1 << 30
        gather, source = entries.to(torch.int32).to(DEV), entries[:rows].clamp(0, tokens - 1).to(DEV)
    else:
        a, sa = (torch.cat([t.view(torch.uint8), t.view(torch.uint8).new_full((extra, t.shape[1]), 255)]).view(t.dtype) for t in (a, sa))
    factor = torch.rand(rows + extra, generator=g).to(DEV) if weighted else None
    got = torch.full((rows + extra, n), 77.0, dtype=out, device=DEV)
    flux_amd.MxGemm(out).forward_grouped(a, torch.tensor(splits, dtype=torch.int32, device=DEV), w, sa, sw, gather_index=gather, row_scale=factor, output=got)
    assert (got[rows:] == 77).all()
    at = 0
    for e, r in enumerate(splits):
        mine = slice(at, at + r)
        check(got[mine], va[source[mine]], vw[e], k, factor[mine] if weighted else None)
        at += r


@pytest.mark.parametrize("few", [0, 1, 40])
def test_far_fewer_rows_than_the_bound(few):
    """The kernel is chosen by the bound of the rows; the splits may leave most of them, or all, unused."""
    for splits, n, k, form in FORMS:
        print(f"[case] {few} rows in form {form} {brief(splits)} {n} {k}", flush=True)
        rows, experts = sum(splits), len(splits)
        few_here = min(few, rows)
        a, sa, va = operand(rows, k=k, seed=1)
        w, sw, vw = operand(experts, n, k=k, seed=2)
        counts = [0] * experts  # the first and the last expert's
        counts[-1] = few_here - few_here // 2
        counts[0] += few_here // 2
        got = torch.full((rows, n), 77.0, device=DEV)
        assert form_of(splits, 0, n, k) == form
        flux_amd.MxGemm(F32).forward_grouped(a, torch.tensor(counts, dtype=torch.int32, device=DEV), w, sa, sw, output=got)
        check(got[:counts[0]], va[:counts[0]], vw[0], k)
        check(got[counts[0]:few_here], va[counts[0]:few_here], vw[-1], k)
        assert (got[few_here:] == 77).all()


@pytest.mark.parametrize("rows,n,k,form", [(5, 300, 640, STREAM), (260, 4095, 640, PANEL), (700, 3001, 1056, PANEL), (3000, 1301, 640, DUAL), (3000, 1301, 2080, DUAL),
                                           (777, 5000, 1024, DUAL), (3000, 1301, 384, TILES), (3000, 1400, 512, TILES)])
def test_every_form_without_splits(rows, n, k, form):
    print(f"[case] dense form {form} {rows} {n} {k}", flush=True)
    assert form_of([rows], 0, n, k)[0] == form
    a, sa, va = operand(rows, k=k, seed=1)
    w, sw, vw = operand(n, k=k, seed=2)
    for out in (BF16, F32):
        check(flux_amd.MxGemm(out).forward(a, w, sa, sw), va, vw, k)


def test_every_form_on_two_streams_at_once():
    """Each call's workspace is its own, and nothing else is shared."""
    calls, seen = [], set()
    for splits, n, k, form in FORMS:
        assert form_of(splits, 0, n, k) == form
        seen.add(form[0])
        a, sa, _ = operand(sum(splits), k=k, seed=1)
        w, sw, _ = operand(len(splits), n, k=k, seed=2)
        sp = torch.tensor(splits, dtype=torch.int32, device=DEV)
        calls.append(lambda a=a, sp=sp, w=w, sa=sa, sw=sw: flux_amd.MxGemm(BF16).forward_grouped(a, sp, w, sa, sw))
    assert seen == {FEW, STREAM, PANEL, DUAL, TILES}
    want = [call() for call in calls]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for which in (0, 1):
            with torch.cuda.stream(streams[which]):
                got[which] += [call() for call in (calls if which else calls[::-1])]
    torch.cuda.synchronize()
    for i, result in enumerate(got[0]):
        assert torch.equal(result, want[-1 - i % len(calls)])
    for i, result in enumerate(got[1]):
        assert torch.equal(result, want[i % len(calls)])


@pytest.mark.parametrize("splits,n,k", [([9, 0, 30], 352, 544), ([300, 257, 0, 700, 65, 512], 1056, 2400)], ids=brief)
def test_gradient_of_the_input_from_the_transposed_codes(splits, n, k):
    """grad_x = grad_y @ W: the weights' transposed codes are the operand whose rows are K, with blocks along N."""
    rows = sum(splits)
    gen = torch.Generator(DEV).manual_seed(n)
    weight = torch.randn(len(splits), n, k, device=DEV, generator=gen).to(BF16)
    grad = torch.randn(rows, n, device=DEV, generator=gen).to(BF16)
    q = quantiser(BF16)
    _, _, codes_t, scale_t = q.quantize_mx(weight, return_tranpose=True)
    gc, gs, _, _ = q.quantize_mx(grad)
    got = flux_amd.MxGemm(F32).forward_grouped(gc, torch.tensor(splits, dtype=torch.int32, device=DEV), codes_t, gs, scale_t)
    assert got.shape == (rows, k)
    vg = torch.from_numpy(mx.values(*mx.quantise(grad.double().cpu().numpy()))).to(DEV)
    at = 0
    for e, r in enumerate(splits):
        vw = torch.from_numpy(mx.values(*mx.quantise(weight[e].t().double().cpu().numpy()))).to(DEV)
        check(got[at:at + r], vg[at:at + r], vw, n)
        at += r


# Streams, both heights of panels, dual tiles and the tiles for short K; counts whose sums pass 2^31, and ones that are twice the rows.
@pytest.mark.parametrize("rows,n,k", [(40, 70, 256), (320, 3001, 512), (800, 3001, 640), (2400, 5000, 1024), (2400, 5000, 1056), (2400, 5000, 384)])
@pytest.mark.parametrize("huge", [1 << 30, (1 << 31) - 1, 0])
def test_counts_far_past_the_rows(rows, n, k, huge):
    """Row counts are on the device, where no check sees them: rows past the last are in no form computed or counted, the experts before have their own."""
    print(f"[case] counts past the rows {rows} {n} {k} {huge}", flush=True)
    a, sa, va = operand(rows, k=k, seed=1)
    w, sw, vw = operand(8, n, k=k, seed=2)
    first, form = rows // 4 + 3, {40: (STREAM, 16), 320: (PANEL, 64), 800: (PANEL, 128)}.get(rows, (TILES if k < 512 else DUAL, 256))
    assert form_of([rows] + [0] * 7, 0, n, k)[:2] == form
    splits = torch.tensor([first, -7, 0, huge or rows, huge or rows, 5, huge or rows, 5], dtype=torch.int32, device=DEV)
    got = flux_amd.MxGemm(F32).forward_grouped(a, splits, w, sa, sw)
    check(got[:first], va[:first], vw[0], k)
    check(got[first:], va[first:], vw[3], k)


@pytest.mark.parametrize("stale", [[0, 0, 40, 0], [1000] * 4, [3, 1, 2, 0]])
def test_row_counts_in_pinned_memory_that_the_stream_has_yet_to_write(stale):
    """A non-blocking copy into the pinned counts is ordered before the call by the stream alone: the call must neither refuse nor use what the host sees in
    them."""
    fresh, n, k = [20, 8, 0, 12], 256, 512
    a, sa, _ = operand(40, k=k, seed=1)
    w, sw, _ = operand(4, n, k=k, seed=2)
    gemm = flux_amd.MxGemm(F32)
    want = gemm.forward_grouped(a, torch.tensor(fresh, dtype=torch.int32), w, sa, sw)
    on_device = torch.tensor(fresh, dtype=torch.int32, device=DEV)
    pinned = torch.empty(4, dtype=torch.int32, pin_memory=True)
    pinned.copy_(torch.tensor(stale, dtype=torch.int32))
    busy = torch.ones(8192, 8192, device=DEV)
    torch.cuda.synchronize()
    for _ in range(4):  # (about 40 ms on the stream)
        torch.mm(busy, busy)
    pinned.copy_(on_device, non_blocking=True)
    got = gemm.forward_grouped(a, pinned, w, sa, sw)
    assert torch.equal(got, want)


def test_gather_entries_past_the_input_are_clamped():
    a, sa, va = operand(6, k=96, seed=1)
    w, sw, vw = operand(1, 33, k=96, seed=2)
    gather = torch.tensor([0, -5, 5, 6, 1 << 30, 3], dtype=torch.int32, device=DEV)
    got = flux_amd.MxGemm(F32).forward_grouped(a, torch.tensor([6], dtype=torch.int32, device=DEV), w, sa, sw, gather_index=gather)
    check(got, va[[0, 0, 5, 5, 5, 3]], vw[0], 96)


@pytest.mark.parametrize("rows,k", [(20, 320), (300, 320), (300, 2048)])
def test_nan_blocks_stay_in_their_rows_and_columns(rows, k):
    a, sa, va = operand(rows, k=k, seed=1)
    w, sw, vw = operand(1, 300, k=k, seed=2)
    sa.view(torch.uint8)[7, 1] = 255
    sw.view(torch.uint8)[0, 50, k // 32 - 1] = 255
    got = flux_amd.MxGemm(F32).forward(a, w[0], sa, sw[0])
    nan = torch.zeros(rows, 300, dtype=torch.bool, device=DEV)
    nan[7], nan[:, 50] = True, True
    assert torch.equal(got.isnan(), nan)
    keep_r, keep_c = [i for i in range(rows) if i != 7], [i for i in range(300) if i != 50]
    check(got[keep_r][:, keep_c], va[keep_r], vw[0][keep_c], k)


def test_no_rows_no_columns():
    a, sa, _ = operand(4, k=64, seed=1)
    w, sw, _ = operand(2, 8, k=64, seed=2)
    gemm = flux_amd.MxGemm(BF16)
    assert gemm.forward(a[:0], w[0], sa[:0], sw[0]).shape == (0, 8)
    assert gemm.forward(a, w[0][:0], sa, sw[0][:0]).shape == (4, 0)
    assert gemm.forward_grouped(a[:0], torch.zeros(2, dtype=torch.int32, device=DEV), w, sa[:0], sw).shape == (0, 8)


def test_weights_past_32_bits():
    experts, n, k = 90, 14336, 7168  # 4.6 GB of codes
    w = torch.randint(0, 256, (experts, n, k // 2), dtype=torch.uint8, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    sw = torch.full((experts, n, k // 32), 120, dtype=torch.uint8, device=DEV)
    a, sa, va = operand(40, k=k, seed=1)
    splits = torch.zeros(experts, dtype=torch.int32)
    splits[0], splits[-1] = 20, 20
    got = flux_amd.MxGemm(F32).forward_grouped(a, splits.to(DEV), w.view(FP4), sa, sw.view(E8M0))
    cols = torch.randint(0, n, (300,), device=DEV)
    q = quantiser(F32)
    for e, rows in ((0, slice(0, 20)), (experts - 1, slice(20, 40))):
        vw = q.dequantize_mx(w[e][cols].view(FP4), sw[e][cols].view(E8M0)).double()
        check(got[rows][:, cols], va[rows], vw, k)


def test_graph_of_a_decode_step_replays():
    """Quantisation and product in one graph, the splits on the device changing between replays."""
    tokens, topk, experts, n, k = 40, 2, 4, 320, 512
    w, sw, _ = operand(experts, n, k=k, seed=2)
    x = torch.randn(tokens, k, device=DEV, dtype=BF16)
    choosed = torch.randint(0, experts, (tokens, topk), dtype=torch.int32, device=DEV)
    q, gemm = quantiser(BF16), flux_amd.MxGemm(BF16)

    def step():
        splits, scatter, gather, _ = flux_amd.moe_route_sort(choosed, experts)
        codes, scale, _, _ = q.quantize_mx(x)
        y = gemm.forward_grouped(codes, splits, w, scale, sw, gather_index=gather)
        return y, flux_amd.moe_unpermute(y, scatter)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for seed in range(4):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        x.copy_(torch.randn(tokens, k, device=DEV, generator=gen))
        choosed.copy_(torch.randint(0, experts - (seed % 2), (tokens, topk), device=DEV, generator=gen))
        want = step()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("pinned", [False, True])
def test_graph_with_row_counts_on_the_host(pinned):
    """A replay reads the counts again from the tensor that the captured call was given."""
    a, sa, _ = operand(40, k=256, seed=1)
    w, sw, _ = operand(4, 70, k=256, seed=2)
    gemm, splits = flux_amd.MxGemm(F32), torch.tensor([10, 0, 25, 5], dtype=torch.int32)
    splits = splits.pin_memory() if pinned else splits
    out = torch.zeros(40, 70, device=DEV)
    gemm.forward_grouped(a, splits, w, sa, sw, output=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gemm.forward_grouped(a, splits, w, sa, sw, output=out)
    for counts in ([10, 0, 25, 5], [1, 2, 3, 4], [40, 0, 0, 0], [0, 0, 0, 0]):
        fresh = torch.tensor(counts, dtype=torch.int32)
        want = torch.full_like(out, 9.0)
        gemm.forward_grouped(a, fresh.to(DEV), w, sa, sw, output=want)
        splits.copy_(fresh)
        out.fill_(9.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_on_another_stream():
    a, sa, va = operand(30, k=640, seed=1)
    w, sw, vw = operand(50, k=640, seed=2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = flux_amd.MxGemm(F32).forward(a, w, sa, sw)
    torch.cuda.current_stream().wait_stream(s)
    check(got, va, vw, 640)


@pytest.mark.parametrize("tokens", [1, 29, 600])
def test_run_of_a_layer(tokens):
    """Tokens to experts, gated MXFP4 products, and back with the router's weights: each step against 64 bits on the outputs of the one before."""
    topk, experts, hidden, ffn = 3, 6, 352, 544
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, hidden, generator=g).to(BF16).to(DEV)
    weight, choosed = torch.topk(torch.softmax(torch.randn(tokens, experts, generator=g), -1).to(DEV), topk)
    choosed = choosed.to(torch.int32)
    q, gemm, gemm32 = quantiser(BF16), flux_amd.MxGemm(BF16), flux_amd.MxGemm(F32)
    (w1, s1, v1), (w3, s3, v3), (w2, s2, v2) = operand(experts, ffn, k=hidden, seed=1), operand(experts, ffn, k=hidden, seed=2), operand(experts, hidden, k=ffn, seed=3)
    splits = torch.bincount(choosed.flatten().long(), minlength=experts).to(torch.int32)
    scatter = flux_amd.calc_scatter_index(choosed, splits)
    # the rows sorted by expert, quantised after the copy or before it: the same codes
    rows = flux_amd.moe_permute(x, scatter)
    codes, scale, _, _ = q.quantize_mx(rows)
    xc, xs, _, _ = q.quantize_mx(x)
    assert torch.equal(flux_amd.moe_permute(xc, scatter).view(torch.uint8), codes.view(torch.uint8))
    assert torch.equal(flux_amd.moe_permute(xs, scatter).view(torch.uint8), scale.view(torch.uint8))
    gate, up = (gemm.forward_grouped(codes, splits, w, scale, s) for w, s in ((w1, s1), (w3, s3)))
    act = torch.nn.functional.silu(gate) * up
    ac, asc, _, _ = q.quantize_mx(act)
    down = gemm32.forward_grouped(ac, splits, w2, asc, s2)
    out = flux_amd.moe_unpermute(down, scatter, weight)
    vx = torch.from_numpy(mx.values(*mx.quantise(rows.double().cpu().numpy()))).to(DEV)
    va = torch.from_numpy(mx.values(*mx.quantise(act.double().cpu().numpy()))).to(DEV)
    at = 0
    for e, r in enumerate(splits.tolist()):
        mine = slice(at, at + r)
        check(gate[mine], vx[mine], v1[e], hidden)
        check(up[mine], vx[mine], v3[e], hidden)
        check(down[mine], va[mine], v2[e], ffn)
        at += r
    terms = down.double()[scatter.long()] * weight.double().unsqueeze(-1)
    assert ((out.double() - terms.sum(1)).abs() <= (topk + 1) * 2.0**-24 * terms.abs().sum(1)).all()


def test_refusals():
    a, sa, _ = operand(4, k=64, seed=1)
    w, sw, _ = operand(2, 8, k=64, seed=2)
    gemm, sp = flux_amd.MxGemm(BF16), torch.tensor([2, 2], dtype=torch.int32, device=DEV)
    q = quantiser(BF16)
    x = torch.zeros(4, 64, dtype=BF16, device=DEV)
    for call, message in (
        (lambda: q.quantize_mx(x.half()), "Inconsistency"),
        (lambda: q.quantize_mx(x.t()), "contiguous"),
        (lambda: q.quantize_mx(x[0]), "2 or 3 dimensions"),
        (lambda: q.quantize_rowwise(x), "float8_e4m3fn"),
        (lambda: q.quantize_vector_blockwise(x), "float8_e4m3fn"),
        (lambda: flux_amd.Quantization(BF16, torch.float8_e4m3fn).quantize_mx(x), "float4_e2m1fn_x2"),
        (lambda: q.dequantize_mx(a, sa, 32), "last of 2 blocks"),
        (lambda: q.dequantize_mx(a, sa, 65), "last of 2 blocks"),
        (lambda: q.dequantize_mx(a, sa[:, :1].contiguous()), "shape mismatch"),
        (lambda: q.dequantize_mx(a.view(torch.uint8), sa), "float4_e2m1fn_x2"),
        (lambda: gemm.forward(a, w[0], sa.view(torch.uint8), sw[0]), "float8_e8m0fnu"),
        (lambda: gemm.forward(a, w[0][:, :16].contiguous(), sa, sw[0][:, :1].contiguous()), "mismatch"),
        (lambda: gemm.forward(a, w, sa, sw), "2 dimensions"),
        (lambda: gemm.forward(a, w[0], sa, sw[0], output=torch.empty(4, 8, device=DEV)), "Inconsistency"),
        (lambda: gemm.forward_grouped(a, sp.long(), w, sa, sw), "int32"),
        (lambda: gemm.forward_grouped(a, sp[:1], w, sa, sw), "splits 0-dim"),
        (lambda: gemm.forward_grouped(a, torch.tensor([3, 2], dtype=torch.int32), w, sa, sw), "sum exceeds"),
        (lambda: gemm.forward_grouped(a, sp, w, sa, sw, row_scale=torch.ones(3, device=DEV)), "row_scale must be"),
        (lambda: gemm.forward_grouped(a, sp, w, sa, sw, gather_index=torch.zeros(4, dtype=torch.int64, device=DEV)), "Inconsistency"),
        (lambda: gemm.forward_grouped(a[:0], sp, w, sa[:0], sw, gather_index=torch.zeros(4, dtype=torch.int32, device=DEV)), "empty input"),
    ):
        with pytest.raises(RuntimeError, match=message):
            call()
