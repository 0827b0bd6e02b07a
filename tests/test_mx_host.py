"""Refusals of the MXFP4 entry points that fire before any HIP call; runs without a GPU."""
import ctypes

import pytest
import torch

import flux_amd
from flux_amd import capi

P, ODD = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1001)


def refused(rc, status, text):
    assert rc == status and text in capi.load().fluxmi_last_error().decode()


def test_quantisation_refuses():
    lib = capi.load()
    refused(lib.fluxmi_quant_mx(P, 3, 1, 4, 64, P, P, None, None, None), -1, "unknown type 3")
    refused(lib.fluxmi_quant_mx(P, 0, -1, 4, 64, P, P, None, None, None), -1, "batch=-1")
    refused(lib.fluxmi_quant_mx(P, 0, 1, -4, 64, P, P, None, None, None), -1, "negative size")
    refused(lib.fluxmi_quant_mx(P, 0, 1, 4, 64, P, P, P, None, None), -1, "go together")
    refused(lib.fluxmi_quant_mx(P, 0, 1, 4, 64, None, P, None, None, None), -1, "null pointer")
    refused(lib.fluxmi_quant_mx(ODD, 0, 1, 4, 64, P, P, None, None, None), -1, "not aligned")
    refused(lib.fluxmi_quant_mx(P, 0, 1, 4, 64, ODD, P, None, None, None), -1, "not aligned")
    refused(lib.fluxmi_quant_mx(P, 0, 1, 4, 64, P, P, ctypes.c_void_p(0x1008), P, None), -1, "not aligned")
    refused(lib.fluxmi_quant_mx(P, 0, 1, 4, 1 << 31, P, P, None, None, None), -2, "exceeds 2^30")
    refused(lib.fluxmi_quant_mx(P, 0, 1, 1 << 40, 64, P, P, None, None, None), -2, "2^40")
    refused(lib.fluxmi_quant_mx(P, 0, 1, 1 << 35, 1, P, P, None, None, None), -2, "more than a launch")
    refused(lib.fluxmi_quant_mx(P, 0, 1, 1 << 31, 32, P, P, P, P, None), -2, "transposed copy")
    assert lib.fluxmi_quant_mx(None, 0, 1, 0, 64, None, None, None, None, None) == 0
    refused(lib.fluxmi_dequant_mx(P, P, 4, 64, 7, P, None), -1, "unknown type 7")
    refused(lib.fluxmi_dequant_mx(P, None, 4, 64, 0, P, None), -1, "null pointer")
    refused(lib.fluxmi_dequant_mx(P, P, 4, 64, 1, ctypes.c_void_p(0x1002), None), -1, "not aligned")


def gemm(**changes):
    fields = dict(nexperts=2, max_rows=8, n=16, k=64, a_rows=8, d_type=0, a=0x1000, a_scale=0x1001, b=0x1000, b_scale=0x1001, d=0x1000, splits=0x1000)
    fields.update(changes)
    return capi.load().fluxmi_grouped_gemm_mx(ctypes.byref(capi.MxGemmArgs(**fields)), None, 0, None)


def test_product_refuses():
    refused(capi.load().fluxmi_grouped_gemm_mx(None, None, 0, None), -1, "null args")
    refused(gemm(nexperts=0), -2, "nexperts=0")
    refused(gemm(nexperts=1025), -2, "nexperts=1025")
    refused(gemm(max_rows=-1), -1, "bad sizes")
    refused(gemm(k=0), -1, "bad sizes")
    refused(gemm(max_rows=(1 << 24) + 1, a_rows=1 << 25, k=32), -2, "exceeds 2^24")
    refused(gemm(splits=None), -1, "null splits")
    refused(gemm(d_type=3), -1, "unknown type 3")
    refused(gemm(n=1 << 20, k=1 << 12), -2, "2 GiB")
    refused(gemm(a_rows=1 << 20, k=1 << 12), -2, "2 GiB")
    refused(gemm(a=None), -1, "null a")
    refused(gemm(b=0x1008), -1, "not 16-byte aligned")
    refused(gemm(d=0x1001), -1, "not 16-byte aligned")
    refused(gemm(a_rows=7), -1, "too few")
    refused(gemm(a_rows=0, gather_a=0x1000), -1, "too few")
    assert gemm(max_rows=0) == 0 and gemm(n=0) == 0


def test_ops_refuse():
    with pytest.raises(RuntimeError, match="bfloat16, float16 or float32"):
        flux_amd.Quantization(torch.float64, torch.float4_e2m1fn_x2)
    with pytest.raises(RuntimeError, match="output dtype"):
        flux_amd.MxGemm(torch.float8_e4m3fn)
    q = flux_amd.Quantization(torch.float16, torch.float4_e2m1fn_x2)
    with pytest.raises(RuntimeError, match="device tensor"):
        q.quantize_mx(torch.zeros(4, 64, dtype=torch.float16))
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        q.quantize_square_blockwise(torch.zeros(4, 64, dtype=torch.float16))
    codes, scale = torch.zeros(4, 32, dtype=torch.uint8).view(torch.float4_e2m1fn_x2), torch.zeros(4, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    with pytest.raises(RuntimeError, match="device tensor"):
        q.dequantize_mx(codes, scale)
    with pytest.raises(RuntimeError, match="device tensor"):
        flux_amd.MxGemm(torch.bfloat16).forward(codes, codes, scale, scale)


def test_forms_and_workspaces():
    """Which kernel computes a product and what it asks for: a copy of the scales where they are not on the words that the kernel reads."""
    def of(*args, **kw):
        info, ws = capi.mx_launch_info(*args, **kw)
        return info.form, info.rows, ws

    def padded(a_rows, b_rows, k):  # scales in rows of whole 16 bytes
        return (a_rows + b_rows) * (((k + 31) // 32 + 15) // 16 * 16)

    assert of(8, 0, 64, 64) == (capi.MX_NONE, 0, 0) and of(8, 64, 0, 64)[0] == capi.MX_NONE
    assert of(2, 8, 300, 705) == (capi.MX_FEW_ROWS, 16, 0)
    assert of(2, 8, 300, 640) == (capi.MX_STREAM, 16, 0) and of(2, 8, 300, 640, scales_at=4) == (capi.MX_STREAM, 16, 0)
    assert of(2, 8, 300, 640, scales_at=1) == (capi.MX_FEW_ROWS, 16, 0)
    assert of(2, 60, 300, 640, scales_at=1) == (capi.MX_STREAM, 32, padded(60, 600, 640)) and of(2, 60, 300, 705) == (capi.MX_STREAM, 32, padded(60, 600, 705))
    assert of(8, 320, 3001, 640) == (capi.MX_PANEL, 64, 0) and of(8, 800, 3001, 640) == (capi.MX_PANEL, 128, 0)
    # 128 experts and K beyond 512 for the dual tiles, which want scales on words only
    assert of(128, 7900, 300, 1408) == (capi.MX_DUAL, 256, 0) and of(129, 7900, 300, 1408) == (capi.MX_TILES, 256, padded(7900, 129 * 300, 1408))
    assert of(129, 7900, 300, 1536) == (capi.MX_TILES, 256, 0) and of(129, 7900, 300, 1536, scales_at=4) == (capi.MX_TILES, 256, padded(7900, 129 * 300, 1536))
    assert of(8, 2000, 2305, 640) == (capi.MX_DUAL, 256, 0) and of(8, 2000, 2305, 512) == (capi.MX_TILES, 256, 0)
    assert of(8, 2000, 2305, 640, a_rows=700, scales_at=2)[2] == padded(700, 8 * 2305, 640)
    # no workspace up to 16 rows per expert, nor for K in 512s with scales on 16 bytes, whatever the sizes
    for experts, n in ((1, 40), (3, 5000), (128, 300), (200, 2048)):
        for k in (96, 705, 1408, 2880):
            for at in (0, 1, 4):
                assert of(experts, 16 * experts, n, k, scales_at=at)[2] == 0
        for rows in (1, 50, 400, 5000, 50000):
            assert of(experts, rows, n, 1536)[2] == 0
    # what the call itself refuses
    lib, info = capi.load(), capi.MxLaunchInfo()
    refused(lib.fluxmi_grouped_gemm_mx_launch_info(None, ctypes.byref(info)), -1, "null args")
    refused(lib.fluxmi_grouped_gemm_mx_launch_info(ctypes.byref(capi.MxGemmArgs()), None), -1, "null args")
    with pytest.raises(RuntimeError, match="exceeds 2\\^24"):
        capi.mx_launch_info(2, (1 << 24) + 1, 16, 32)
    with pytest.raises(RuntimeError, match="nexperts=0"):
        capi.mx_launch_info(0, 8, 16, 32)
