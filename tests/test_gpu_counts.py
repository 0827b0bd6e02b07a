"""Row counts on the device that exceed the rows: every form of the grouped GEMM computes what the counts name up to the last row, and no sum of them overflows.

The results are compared with those of the counts cut to the rows, bit for bit: the schedule sees the same experts, rows and tiles."""
import pytest
import torch

from flux_amd import capi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn
# generic, streams, panels, macro tiles, dual tiles, and launches of two forms between which the counts decide
SIZES = [(8, 60, 34, 72, capi.GEMM_GENERIC), (8, 12, 512, 8192, capi.GEMM_STREAM), (8, 40, 256, 512, capi.GEMM_PANEL), (8, 800, 4096, 1024, capi.GEMM_PANEL),
         (8, 2400, 2048, 1024, capi.GEMM_MACRO_TILES), (8, 8000, 2048, 4096, capi.GEMM_MACRO_TILES), (70, 2000, 512, 512, capi.GEMM_BY_SPLITS),
         (70, 140, 256, 4096, capi.GEMM_BY_SPLITS), (200, 9000, 256, 512, capi.GEMM_BY_SPLITS)]


def cut(counts, rows):
    out = []
    for c in counts:
        out.append(min(max(c, 0), rows - sum(out)))
    return out


def patterns(experts, rows):
    first, huge, most = rows // 3 + 1, 1 << 30, (1 << 31) - 1
    rest = [0, 5] * ((experts - 5) // 2) + [7] * ((experts - 5) % 2)
    return ([first, -7, huge, huge, 5] + rest, [huge] * experts, [0, most, most, 1, most] + rest, [first, rows, rows, -(1 << 31), 2] + rest,
            [1] * (experts - 2) + [most, most])


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("experts,rows,n,k,form", SIZES)
def test_counts_past_the_rows(experts, rows, n, k, form, dtype):
    print(f"[case] counts {experts} {rows} {n} {k} {dtype}", flush=True)
    assert capi.gemm_launch_info(dtype, experts, rows, n, k).form == form
    g = torch.Generator(DEV).manual_seed(n)
    x = torch.randn(rows, k, device=DEV, generator=g).to(dtype)
    w = (torch.randn(experts, n, k, device=DEV, generator=g) * 0.05).to(dtype)
    for counts in patterns(experts, rows):
        device = lambda c: torch.tensor(c, dtype=torch.int32, device=DEV)  # noqa: E731
        want = capi.grouped_gemm(x, w, device(cut(counts, rows)), out=torch.full((rows, n), 77.0, dtype=BF16, device=DEV))
        got = capi.grouped_gemm(x, w, device(counts), out=torch.full((rows, n), 77.0, dtype=BF16, device=DEV))
        assert torch.equal(got, want)


@pytest.mark.parametrize("experts,rows,n,k", [(8, 40, 256, 512), (8, 800, 1024, 1024), (8, 4000, 1024, 512), (70, 2000, 512, 512)])
def test_counts_past_the_rows_block_scaled(experts, rows, n, k):
    print(f"[case] counts, block scales {experts} {rows} {n} {k}", flush=True)
    g = torch.Generator(DEV).manual_seed(n)
    x, w = torch.randn(rows, k, device=DEV, generator=g).to(FP8), (torch.randn(experts, n, k, device=DEV, generator=g) * 0.05).to(FP8)
    a_scale = torch.rand((rows + 127) // 128, k // 128, 128, device=DEV, generator=g) + 0.5
    b_scale = torch.rand(experts, n // 128, k // 128, device=DEV, generator=g) + 0.5
    for counts in patterns(experts, rows):
        device = lambda c: torch.tensor(c, dtype=torch.int32, device=DEV)  # noqa: E731
        want = capi.grouped_gemm_blockscale(x, w, device(cut(counts, rows)), a_scale, b_scale, out=torch.full((rows, n), 77.0, dtype=BF16, device=DEV))
        got = capi.grouped_gemm_blockscale(x, w, device(counts), a_scale, b_scale, out=torch.full((rows, n), 77.0, dtype=BF16, device=DEV))
        assert torch.equal(got, want)
