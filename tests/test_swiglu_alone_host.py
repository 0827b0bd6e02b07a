"""fluxmi_swiglu_backward without a gradient: what is refused before any HIP call; runs without a GPU."""
import ctypes

from flux_amd import capi

P, Q = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x2000)


def test_the_activation_alone_needs_its_result_and_no_gradient():
    lib = capi.load()
    for grad, grad_x, out in ((None, None, None), (None, Q, P), (P, None, Q)):
        rc = lib.fluxmi_swiglu_backward(grad, P, None, 0, 4, 64, grad_x, out, None)
        assert rc == -1 and "null pointer" in lib.fluxmi_last_error().decode()
