"""What the experts' layers record: gradients that are not lost, and backward passes that compute and keep what is asked for alone."""
import pytest
import torch

import flux_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16 = torch.bfloat16, torch.float16


def data(shape, dtype, seed, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(DEV)


def counts(splits):
    return torch.tensor(splits, dtype=torch.int32, device=DEV)


def same(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 33), (70, 256), (0, 64)])
def test_swiglu_checkpoint_has_the_activations_gradient(rows, cols, dtype):
    x, up = data((rows, 2 * cols), dtype, 1, 2.0).requires_grad_(), data((rows, cols), dtype, 2)
    out, codes, scale = flux_amd.moe_swiglu_checkpoint(x)
    assert out.requires_grad and not codes.requires_grad and not scale.requires_grad
    plain = flux_amd.moe_swiglu_checkpoint(x.detach())
    assert same(out.detach(), plain[0]) and same(codes, plain[1]) and same(scale, plain[2]) and not plain[0].requires_grad
    out.backward(up)
    assert torch.equal(x.grad, flux_amd.moe_swiglu_backward(up, codes, scale)[0])
    other = x.detach().clone().requires_grad_()
    flux_amd.moe_swiglu(other, checkpoint=True).backward(up)
    assert torch.equal(x.grad, other.grad)
    with torch.no_grad():
        assert not flux_amd.moe_swiglu_checkpoint(x)[0].requires_grad


def test_swiglu_checkpoint_between_two_products():
    """By hand in grad mode: the first weights' gradient is there."""
    splits = counts([20, 0, 13])
    x, w1, w2 = data((33, 64), BF16, 1), data((3, 96, 64), BF16, 2, 0.1).requires_grad_(), data((3, 64, 48), BF16, 3, 0.1).requires_grad_()
    out, _, _ = flux_amd.moe_swiglu_checkpoint(flux_amd.moe_linear(x, w1, splits))
    up = data((33, 64), BF16, 4)
    flux_amd.moe_linear(out, w2, splits).backward(up)
    a, b = w1.detach().clone().requires_grad_(), w2.detach().clone().requires_grad_()
    flux_amd.moe_linear(flux_amd.moe_swiglu(flux_amd.moe_linear(x, a, splits), checkpoint=True), b, splits).backward(up)
    assert torch.equal(w1.grad, a.grad) and torch.equal(w2.grad, b.grad) and w1.grad.any()


def test_swiglu_checkpoint_refuses_what_the_activation_refuses():
    x = data((4, 64), BF16, 1).requires_grad_()
    with pytest.raises(RuntimeError, match="gradient of the gradient"):
        torch.autograd.grad(flux_amd.moe_swiglu_checkpoint(x)[0].sum(), [x], create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            flux_amd.moe_swiglu_checkpoint(torch.autograd.forward_ad.make_dual(x.detach(), x.detach()))
    alive = flux_amd.moe_swiglu(x)
    with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            flux_amd.moe_swiglu_checkpoint(x)[0].sum().backward()
    del alive
