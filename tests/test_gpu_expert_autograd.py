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


# ---- the second weights alone ---------------------------------------------------------------------------------------


def mlp_operands(splits, rest, hidden, ffn, dtype):
    return (data((sum(splits) + rest, hidden), dtype, 1), data((len(splits), 2 * ffn, hidden), dtype, 2, hidden**-0.5), data((len(splits), hidden, ffn), dtype, 3, ffn**-0.5))


@pytest.mark.parametrize("ckpt", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("splits,rest,hidden,ffn", [([20, 0, 11], 3, 64, 33), ([300, 70], 0, 128, 160), ([0, 0], 2, 8, 8)])
def test_second_weights_alone(splits, rest, hidden, ffn, dtype, ckpt):
    """Their gradient has the bits of a pass over everything, and the pass neither reads nor keeps the weights: they may change in between."""
    x, w1, w2 = mlp_operands(splits, rest, hidden, ffn, dtype)
    up = data((x.shape[0], hidden), dtype, 4)
    whole = [t.clone().requires_grad_() for t in (x, w1, w2)]
    flux_amd.moe_mlp(*whole, counts(splits), checkpoint=ckpt).backward(up)
    alone = w2.clone().requires_grad_()
    out = flux_amd.moe_mlp(x, w1, alone, counts(splits), checkpoint=ckpt)
    with torch.no_grad():
        alone.mul_(2)
    out.backward(up)
    assert torch.equal(alone.grad, whole[2].grad)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (129, 2047), (40, 96)])
def test_the_activation_alone(rows, cols, dtype):
    """The C entry without a gradient: the bits that come beside one, and nothing else is written."""
    from flux_amd import capi

    x = data((rows, 2 * cols), dtype, 1, 3.0)
    out, codes, scale = flux_amd.moe_swiglu_checkpoint(x)
    grad = data((rows, cols), dtype, 2)
    for given, its_scale in ((x, None), (codes, scale)):
        want = flux_amd.moe_swiglu_backward(grad, given, its_scale)[1]
        flat = torch.full((rows * cols + 16,), 7.0, dtype=dtype, device=DEV)
        rc = capi.load().fluxmi_swiglu_backward(None, capi._ptr(given), capi._ptr(its_scale), capi._ROW_TYPES[dtype], rows, cols, None, capi._ptr(flat), capi._stream())
        assert rc == 0 and torch.equal(flat[:rows * cols].view(rows, cols), want) and (flat[rows * cols:] == 7).all()


# ---- backward passes that are asked for some of the gradients -------------------------------------------------------


def allocated(call):
    """A call's result, and the bytes that it allocated, freed ones among them."""
    before = torch.cuda.memory_stats()["allocated_bytes.all.allocated"]
    result = call()
    return result, torch.cuda.memory_stats()["allocated_bytes.all.allocated"] - before


@pytest.mark.parametrize("ckpt", [False, True])
def test_gradients_that_are_not_asked_for_are_not_computed(ckpt):
    """A weights' gradient that is left out leaves out its memory."""
    splits, hidden, ffn = [5, 0, 9, 2], 512, 1024
    leaves = [t.requires_grad_() for t in mlp_operands(splits, 0, hidden, ffn, BF16)]
    x, w1, w2 = leaves
    up, up1 = data((16, hidden), BF16, 4), data((16, 2 * ffn), BF16, 5)
    out = flux_amd.moe_mlp(*leaves, counts(splits), checkpoint=ckpt)
    whole, all_bytes = allocated(lambda: torch.autograd.grad(out, leaves, up))
    for wanted in range(1, 7):
        some = [i for i in range(3) if wanted >> i & 1]
        out = flux_amd.moe_mlp(*leaves, counts(splits), checkpoint=ckpt)
        got, its_bytes = allocated(lambda: torch.autograd.grad(out, [leaves[i] for i in some], up))
        assert all(torch.equal(g, whole[i]) for g, i in zip(got, some))
        assert its_bytes <= all_bytes - sum(t.numel() * 2 for i, t in enumerate(leaves) if i not in some)
    out = flux_amd.moe_linear(x, w1, counts(splits), ckpt)
    whole, all_bytes = allocated(lambda: torch.autograd.grad(out, [x, w1], up1))
    for i, leaf in enumerate((x, w1)):
        out = flux_amd.moe_linear(x, w1, counts(splits), ckpt)
        got, its_bytes = allocated(lambda: torch.autograd.grad(out, [leaf], up1))
        assert torch.equal(got[0], whole[i]) and its_bytes <= all_bytes - (w1 if i == 0 else x).numel() * 2


def test_a_frozen_layer_before_one_that_learns():
    """Gradients of intermediate results, of a graph in which some leaves want none, and of one leaf used twice."""
    splits = counts([20, 13])
    x, w1, w2 = mlp_operands([20, 13], 0, 64, 32, BF16)
    x.requires_grad_()
    middle = x * 2
    out = flux_amd.moe_mlp(middle, w1, w2, splits)
    up = data(out.shape, BF16, 4)
    of_middle, = torch.autograd.grad(out, [middle], up, retain_graph=True)
    of_x, = torch.autograd.grad(out, [x], up)
    assert torch.equal(of_x, of_middle * 2)
    w = data((2, 64, 64), BF16, 5, 0.1).requires_grad_()
    y = flux_amd.moe_linear(flux_amd.moe_linear(x, w, splits), w, splits)
    a, b = torch.autograd.grad(y, [x, w], up, retain_graph=True)
    assert torch.equal(torch.autograd.grad(y, [w], up, retain_graph=True)[0], b) and torch.equal(torch.autograd.grad(y, [x], up)[0], a)
