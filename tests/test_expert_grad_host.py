"""Refusals of the entry points of the experts' gradients that fire before any HIP call; runs without a GPU."""
import ctypes

import pytest
import torch

import flux_amd
from flux_amd import capi

P, Q = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x2000)
ODD = ctypes.c_void_p(0x1001)


def refused(rc, status, text):
    assert rc == status and text in capi.load().fluxmi_last_error().decode(), capi.load().fluxmi_last_error()


def test_c_entry_points_refuse():
    lib = capi.load()
    dgrad = lambda grad=P, weight=P, t=0, splits=P, e=2, rows=4, n=64, k=64, out=Q, ws=None, ws_bytes=0: lib.fluxmi_moe_dgrad(grad, weight, t, splits, e, rows, n, k, out, ws, ws_bytes, None)  # noqa: E731
    refused(dgrad(t=1), -1, "type 1")
    refused(dgrad(e=-1), -1, "negative")
    refused(dgrad(rows=-4), -1, "negative")
    refused(dgrad(e=1025), -2, "nexperts=1025")
    refused(dgrad(rows=(1 << 24) + 1), -2, "at most 2^24")
    refused(dgrad(n=(1 << 24) + 1), -2, "over 2^24")
    refused(dgrad(rows=1 << 24, k=1 << 24), -2, "too many")
    refused(dgrad(grad=None), -1, "null pointer")
    refused(dgrad(splits=None), -1, "null pointer")
    refused(dgrad(grad=ODD), -1, "aligned")
    refused(dgrad(out=ctypes.c_void_p(0x1002)), -1, "aligned")
    need = lib.fluxmi_moe_dgrad_workspace_bytes(2, 4, 4096, 64)
    assert need > 0
    refused(dgrad(n=4096, ws=P, ws_bytes=need - 1), -3, "workspace")
    refused(dgrad(n=4096, ws=ctypes.c_void_p(0x1004), ws_bytes=need), -3, "workspace")
    assert lib.fluxmi_moe_dgrad_workspace_bytes(-1, 4, 4096, 64) == 0 and lib.fluxmi_moe_dgrad_workspace_bytes(0, 0, 0, 0) == 0
    assert dgrad(rows=0, grad=None, out=None) == 0 and dgrad(k=0, out=None) == 0

    wgrad = lambda grad=P, x=P, scale=None, t=0, splits=P, e=2, rows=4, n=64, k=64, out=Q, out_t=0, ws=None, ws_bytes=0: lib.fluxmi_moe_wgrad(  # noqa: E731
        grad, x, scale, t, splits, e, rows, n, k, out, out_t, 0, ws, ws_bytes, None)
    refused(wgrad(t=3), -1, "type 3")
    refused(wgrad(out_t=2), -1, "out_type 2")
    refused(wgrad(x=None), -1, "null pointer")
    refused(wgrad(out=None), -1, "null pointer")
    refused(wgrad(x=ODD), -1, "aligned")
    refused(wgrad(out=ctypes.c_void_p(0x1008)), -1, "aligned")
    refused(wgrad(e=1000, n=1 << 20, k=1 << 20), -2, "too many")
    need = lib.fluxmi_moe_wgrad_workspace_bytes(2, 100000, 64, 64)
    assert need > 0
    refused(wgrad(rows=100000, ws=P, ws_bytes=need - 1), -3, "workspace")
    refused(wgrad(rows=100000), -3, "workspace")
    refused(wgrad(rows=100000, ws=ctypes.c_void_p(0x1004), ws_bytes=need), -3, "workspace")
    assert wgrad(e=0, out=None) == 0 and wgrad(k=0, out=None) == 0
    assert lib.fluxmi_moe_wgrad_workspace_bytes(-1, 100000, 64, 64) == 0 and lib.fluxmi_moe_wgrad_workspace_bytes(0, 0, 0, 0) == 0

    refused(lib.fluxmi_moe_clear_rest(P, P, 2, 4, -1, None), -1, "row_bytes")
    refused(lib.fluxmi_moe_clear_rest(None, P, 2, 4, 8, None), -1, "null pointer")
    refused(lib.fluxmi_moe_clear_rest(P, ODD, 2, 4, 8, None), -1, "not 4-byte aligned")
    refused(lib.fluxmi_checkpoint_e4m3(P, 1, 4, 64, P, P, None), -1, "type 1")
    refused(lib.fluxmi_checkpoint_e4m3(P, 0, -4, 64, P, P, None), -1, "negative")
    refused(lib.fluxmi_checkpoint_e4m3(P, 0, 4, 1 << 31, P, P, None), -2, "2^30 columns")
    refused(lib.fluxmi_checkpoint_e4m3(P, 0, 1 << 40, 64, P, P, None), -2, "too many rows")
    refused(lib.fluxmi_checkpoint_e4m3(ODD, 0, 4, 64, P, P, None), -1, "aligned")
    refused(lib.fluxmi_checkpoint_e4m3(P, 0, 4, 64, None, P, None), -1, "null pointer")
    assert lib.fluxmi_checkpoint_e4m3(None, 0, 0, 64, None, None, None) == 0
    refused(lib.fluxmi_swiglu(P, 0, 4, 64, P, P, None, None), -1, "come together")
    refused(lib.fluxmi_swiglu(P, 0, 4, 64, None, None, None, None), -1, "null pointer")
    refused(lib.fluxmi_swiglu_backward(P, P, None, 0, 4, 64, None, P, None), -1, "null pointer")
    refused(lib.fluxmi_swiglu_backward(P, ODD, None, 0, 4, 64, P, P, None), -1, "aligned")


def calls(x, w, w2, splits, e4m3, e8m0):
    return {"moe_linear": lambda: flux_amd.moe_linear(x, w, splits), "moe_swiglu": lambda: flux_amd.moe_swiglu(x),
            "moe_mlp": lambda: flux_amd.moe_mlp(x, w, w2, splits), "moe_dgrad": lambda: flux_amd.moe_dgrad(x, w2, splits),
            "moe_wgrad": lambda: flux_amd.moe_wgrad(x, x, splits), "moe_wgrad of 8 bits": lambda: flux_amd.moe_wgrad(x, e4m3, splits, e8m0),
            "moe_checkpoint": lambda: flux_amd.moe_checkpoint(x), "moe_swiglu_checkpoint": lambda: flux_amd.moe_swiglu_checkpoint(x),
            "moe_swiglu_backward": lambda: flux_amd.moe_swiglu_backward(x, x)}


def operands(make=lambda t: t):
    bf16 = torch.bfloat16
    return calls(make(torch.zeros(4, 8, dtype=bf16)), torch.zeros(2, 16, 8, dtype=bf16), torch.zeros(2, 8, 8, dtype=bf16), torch.zeros(2, dtype=torch.int32),
                 torch.zeros(4, 8, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu))


def test_ops_refuse_host_tensors():
    for name, call in operands().items():
        with pytest.raises(RuntimeError, match="device tensor"):
            call()
            pytest.fail(name)


def test_tangents_are_refused():
    with torch.autograd.forward_ad.dual_level():
        for name, call in operands(lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))).items():
            with pytest.raises(RuntimeError, match="forward-mode derivatives"):
                call()
                pytest.fail(name)


def test_negative_views_are_refused():
    for name, call in operands(torch._neg_view).items():
        with pytest.raises(RuntimeError, match="conjugate or negative view"):
            call()
            pytest.fail(name)
