"""Refusals of the expert permutation's entry points that fire before any HIP call; runs without a GPU."""
import ctypes

import pytest
import torch

import flux_amd
from flux_amd import capi

P = ctypes.c_void_p(0x1000)
ODD = ctypes.c_void_p(0x1001)


def refused(rc, status, text):
    assert rc == status and text in capi.load().fluxmi_last_error().decode()


def test_c_entry_points_refuse():
    lib = capi.load()
    refused(lib.fluxmi_moe_permute(P, P, -1, 2, 64, P, None), -1, "negative ntokens")
    refused(lib.fluxmi_moe_permute(P, P, 4, 0, 64, P, None), -2, "topk=0")
    refused(lib.fluxmi_moe_permute(P, P, 4, 65, 64, P, None), -2, "topk=65")
    refused(lib.fluxmi_moe_permute(P, P, 1 << 30, 2, 64, P, None), -2, "exceeds 2^30")
    refused(lib.fluxmi_moe_permute(P, None, 4, 2, 64, P, None), -1, "null scatter_index")
    refused(lib.fluxmi_moe_permute(P, ODD, 4, 2, 64, P, None), -1, "not 4-byte aligned")
    refused(lib.fluxmi_moe_permute(None, P, 4, 2, 64, P, None), -1, "null pointer")
    refused(lib.fluxmi_moe_permute(P, P, 4, 2, -1, P, None), -1, "row_bytes")
    refused(lib.fluxmi_moe_permute(P, P, 1 << 30, 1, 16, P, None), -2, "too many")
    assert lib.fluxmi_moe_permute(None, None, 0, 2, 64, None, None) == 0
    refused(lib.fluxmi_moe_unpermute(P, 3, P, None, 1, 4, 2, 64, P, None), -1, "unknown type 3")
    refused(lib.fluxmi_moe_unpermute(P, 0, P, P, 9, 4, 2, 64, P, None), -1, "unknown type 9")
    refused(lib.fluxmi_moe_unpermute(ODD, 0, P, P, 1, 4, 2, 64, P, None), -1, "not aligned")
    refused(lib.fluxmi_moe_unpermute(P, 0, P, P, 1, 4, 2, -8, P, None), -1, "negative n")
    refused(lib.fluxmi_moe_unpermute(P, 0, P, P, 1, 4, 2, 64, None, None), -1, "null pointer")
    refused(lib.fluxmi_moe_unpermute_backward(P, P, 0, P, None, 1, 4, 2, 64, P, P, None), -1, "null pointer")
    refused(lib.fluxmi_moe_unpermute_backward(P, None, 0, P, P, 1, 4, 2, 64, P, P, None), -1, "null pointer")
    refused(lib.fluxmi_moe_unpermute_backward(P, P, 0, P, P, 1, 4, 2, 64, None, None, None), -1, "null pointer")
    refused(lib.fluxmi_moe_unpermute_backward(P, P, 1, P, P, 1, 4, 2, 64, ctypes.c_void_p(0x1002), P, None), -1, "not aligned")


def test_ops_refuse_host_tensors():
    idx = torch.zeros(4, 2, dtype=torch.int32)
    for call in (lambda: flux_amd.moe_permute(torch.zeros(4, 8), idx), lambda: flux_amd.moe_permute_backward(torch.zeros(8, 8), idx),
                 lambda: flux_amd.moe_unpermute(torch.zeros(8, 8), idx, torch.ones(4, 2)),
                 lambda: flux_amd.moe_unpermute_backward(torch.zeros(4, 8), torch.zeros(8, 8), idx, torch.ones(4, 2))):
        with pytest.raises(RuntimeError, match="device tensor"):
            call()


def test_tangents_are_refused():
    """Forward mode: a dual tensor that requires no gradient would come back without its tangent."""
    idx, x, rows, w = torch.zeros(4, 2, dtype=torch.int32), torch.ones(4, 8), torch.ones(8, 8), torch.ones(4, 2)
    with torch.autograd.forward_ad.dual_level():
        dx, drows = (torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, rows))
        for call in (lambda: flux_amd.moe_permute(dx, idx), lambda: flux_amd.moe_permute_backward(drows, idx), lambda: flux_amd.moe_unpermute(drows, idx),
                     lambda: flux_amd.moe_unpermute(drows, idx, w), lambda: flux_amd.moe_unpermute_backward(dx, rows, idx, w)):
            with pytest.raises(RuntimeError, match="forward-mode derivatives"):
                call()


def test_conjugate_and_negative_views_are_refused():
    """Their memory holds other values than they stand for, and rows are moved as memory."""
    idx, w = torch.zeros(4, 2, dtype=torch.int32), torch.ones(4, 2)
    conj, neg, neg_rows = torch.ones(4, 8, dtype=torch.complex64).conj(), torch._neg_view(torch.ones(4, 8)), torch._neg_view(torch.ones(8, 8))
    for call in (lambda: flux_amd.moe_permute(conj, idx), lambda: flux_amd.moe_permute(neg, idx), lambda: flux_amd.moe_permute_backward(neg_rows, idx),
                 lambda: flux_amd.moe_unpermute(neg_rows, idx, w), lambda: flux_amd.moe_unpermute_backward(neg, torch.ones(8, 8), idx, w)):
        with pytest.raises(RuntimeError, match="conjugate or negative view"):
            call()
