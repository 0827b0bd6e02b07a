"""moe_permute, moe_unpermute and their backward passes against the formulas in 64 bits.

Bounds: a copied row is exact.  A sum of k products in fp32 is off by at most k + 1 roundings of 2^-24 of the sum of magnitudes, and its result is
rounded once to the rows' type (half a step, eps / 2 of the value).  A weight's gradient sums n products, at least eight lanes share
them: chains of at most n / 8 + 16 roundings."""
import pytest
import torch

import flux_amd
from flux_amd import capi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make_index(tokens, topk, dropped, seed, experts=8, shuffled=False):
    """A stable sort's index with a share of dropped pairs; shuffled: any distinct rows, with holes where pairs are dropped."""
    g = torch.Generator().manual_seed(seed)
    pairs = tokens * topk
    lost = torch.rand(pairs, generator=g) < dropped
    if shuffled:
        idx = torch.randperm(pairs, generator=g)
    else:
        expert = torch.where(lost, experts, torch.randint(0, experts, (pairs,), generator=g))
        order = torch.argsort(expert, stable=True)
        idx = torch.empty_like(order)
        idx[order] = torch.arange(pairs)
    return torch.where(lost, -1, idx).to(torch.int32).view(tokens, topk).to(DEV)


def data(rows, cols, dtype, seed):
    return torch.randn(rows, cols, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def want_rows(per_token, idx, scale=None):
    """fp64 rows [pairs, n]: rows[idx[t, j]] = scale[t, j] * per_token[t]."""
    tokens, topk = idx.shape
    out = torch.zeros(tokens * topk, per_token.shape[1], dtype=torch.float64, device=DEV)
    named = idx >= 0
    token = torch.arange(tokens, device=DEV)[:, None].expand_as(idx)[named]
    v = per_token.double()[token]
    out[idx[named].long()] = v if scale is None else v * scale.double()[named][:, None]
    return out


def pair_rows(rows, idx):
    """fp64 [tokens, topk, n], zeros for dropped pairs."""
    padded = torch.cat([rows.double(), rows.new_zeros(1, rows.shape[1]).double()])
    return padded[torch.where(idx >= 0, idx.long(), rows.shape[0])]


def close(got, want, magnitude, roundings):
    half_step = torch.finfo(got.dtype).eps / 2 if got.dtype != F32 else 0.0
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps  # half a step of subnormal results
    bound = half_step * want.abs() + roundings * 2.0**-24 * magnitude + tiny
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= bound * 1.0000001).all(), f"off by {(off - bound).max().item():.3g} more than the bound"


SHAPES = [(1, 1, 1), (1, 2, 7), (3, 1, 8), (5, 3, 9), (37, 2, 4096), (64, 6, 31), (129, 8, 2047), (300, 4, 1024), (1000, 9, 96), (2, 64, 257),
          (513, 2, 7168), (5000, 2, 40), (7, 5, 16384)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,topk,n", SHAPES)
@pytest.mark.parametrize("dropped,shuffled", [(0.0, False), (0.3, False), (0.3, True)])
def test_permute_copies_rows_and_clears_the_others(tokens, topk, n, dtype, dropped, shuffled):
    print(f"[case] permute {tokens} {topk} {n} {dtype} {dropped} {shuffled}", flush=True)
    idx, x = make_index(tokens, topk, dropped, n, shuffled=shuffled), data(tokens, n, dtype, 1)
    want = want_rows(x, idx)
    dirty = torch.full((tokens * topk, n), float("nan"), dtype=dtype, device=DEV)
    assert torch.equal(capi.moe_permute(x, idx, out=dirty).double(), want)
    assert torch.equal(flux_amd.moe_permute(x, idx).double(), want)


@pytest.mark.parametrize("wtype", [None, F32, "same"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,topk,n", SHAPES)
def test_unpermute(tokens, topk, n, dtype, wtype):
    print(f"[case] unpermute {tokens} {topk} {n} {dtype} {wtype}", flush=True)
    idx, rows = make_index(tokens, topk, 0.2, n + 1), data(tokens * topk, n, dtype, 2)
    rows[int((idx >= 0).sum()):] = float("nan")  # rows that no pair names are not read
    w = None if wtype is None else torch.rand(tokens, topk, generator=torch.Generator().manual_seed(3)).to(dtype if wtype == "same" else F32).to(DEV)
    terms = pair_rows(rows, idx).nan_to_num()
    if w is not None:
        terms = terms * w.double().unsqueeze(-1)
    got = flux_amd.moe_unpermute(rows, idx, w)
    close(got, terms.sum(1), terms.abs().sum(1), topk + 1)
    assert torch.equal(got, capi.moe_unpermute(rows, idx, w))
    if w is None:
        assert torch.equal(got, flux_amd.moe_permute_backward(rows, idx))


@pytest.mark.parametrize("wtype", [F32, "same"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,topk,n", SHAPES)
def test_unpermute_backward(tokens, topk, n, dtype, wtype):
    print(f"[case] unpermute_backward {tokens} {topk} {n} {dtype} {wtype}", flush=True)
    idx, rows, grad = make_index(tokens, topk, 0.2, n + 2), data(tokens * topk, n, dtype, 4), data(tokens, n, dtype, 5)
    w = torch.rand(tokens, topk, generator=torch.Generator().manual_seed(6)).to(dtype if wtype == "same" else F32).to(DEV)
    grad_rows, grad_w = flux_amd.moe_unpermute_backward(grad, rows, idx, w)
    assert grad_rows.dtype == dtype and grad_w.dtype == w.dtype
    want = want_rows(grad, idx, w)
    close(grad_rows, want, want.abs(), 1)
    products = pair_rows(rows, idx) * grad.double().unsqueeze(1)
    close(grad_w, products.sum(-1), products.abs().sum(-1), n / 8 + 16)
    assert (grad_w[idx < 0] == 0).all()


@pytest.mark.parametrize("offset", [1, 3])
def test_rows_at_any_element(offset):
    """Rows that start between vectors, as a slice of a larger buffer does."""
    tokens, topk, n = 33, 3, 129
    idx = make_index(tokens, topk, 0.1, 7)
    for dtype in (BF16, F32):
        def at(rows, seed):
            flat = torch.zeros(rows * n + offset, dtype=dtype, device=DEV)
            flat[offset:] = data(rows, n, dtype, seed).flatten()
            return flat[offset:].view(rows, n)
        x, rows, w = at(tokens, 8), at(tokens * topk, 9), torch.rand(tokens, topk, device=DEV)
        assert torch.equal(flux_amd.moe_permute(x, idx), flux_amd.moe_permute(x.clone(), idx))
        assert torch.equal(flux_amd.moe_unpermute(rows, idx, w), flux_amd.moe_unpermute(rows.clone(), idx, w))
        a, b = flux_amd.moe_unpermute_backward(x, rows, idx, w), flux_amd.moe_unpermute_backward(x.clone(), rows.clone(), idx, w)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # an index that does not start on 16 bytes
    flat = torch.full((tokens * topk + offset,), -1, dtype=torch.int32, device=DEV)
    flat[offset:] = idx.flatten()
    assert torch.equal(flux_amd.moe_permute(x, flat[offset:].view(tokens, topk)), flux_amd.moe_permute(x, idx))


def test_rows_of_bytes():
    """Codes and scales of quantised tokens go the same way: any type, odd widths."""
    idx = make_index(50, 2, 0.1, 11)
    for n in (1, 15, 33, 448):
        x = torch.randint(0, 256, (50, n), dtype=torch.uint8, device=DEV)
        for t in (torch.uint8, torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.float4_e2m1fn_x2):
            got = flux_amd.moe_permute(x.view(t), idx)
            assert got.dtype == t and torch.equal(got.view(torch.uint8).double(), want_rows(x, idx))


def test_no_tokens_no_columns_no_pairs():
    e = torch.empty
    idx0, idx = e(0, 2, dtype=torch.int32, device=DEV), make_index(5, 2, 0.0, 1)
    assert flux_amd.moe_permute(e(0, 16, device=DEV), idx0).shape == (0, 16)
    assert flux_amd.moe_unpermute(e(0, 16, device=DEV), idx0).shape == (0, 16)
    assert flux_amd.moe_permute(e(5, 0, device=DEV), idx).shape == (10, 0)
    a, b = flux_amd.moe_unpermute_backward(e(5, 0, device=DEV), e(10, 0, device=DEV), idx, torch.ones(5, 2, device=DEV))
    assert a.shape == (10, 0) and (b == 0).all()
    none = torch.full((5, 2), -1, dtype=torch.int32, device=DEV)
    x = data(5, 16, F32, 1)
    assert (flux_amd.moe_permute(x, none) == 0).all() and (flux_amd.moe_unpermute(flux_amd.moe_permute(x, none), none) == 0).all()
    a, b = flux_amd.moe_unpermute_backward(x, data(10, 16, F32, 2), none, torch.ones(5, 2, device=DEV))
    assert (a == 0).all() and (b == 0).all()


def test_infinities_stay_in_their_rows():
    idx = torch.tensor([[0, 1], [2, -1]], dtype=torch.int32, device=DEV)
    rows = torch.ones(4, 64, device=DEV)
    rows[1, 5], rows[3] = float("inf"), float("nan")
    w = torch.tensor([[1.0, 0.5], [2.0, float("nan")]], device=DEV)  # the dropped pair's weight is not used
    out = flux_amd.moe_unpermute(rows, idx, w)
    assert out[0, 5] == float("inf") and torch.isfinite(out[0, :5]).all() and (out[1] == 2).all()
    grad_rows, grad_w = flux_amd.moe_unpermute_backward(torch.ones(2, 64, device=DEV), rows, idx, w)
    assert (grad_rows[3] == 0).all() and (grad_rows[2] == 2).all()
    assert grad_w[0, 0] == 64 and grad_w[0, 1] == float("inf") and grad_w[1, 0] == 64 and grad_w[1, 1] == 0


def test_offsets_past_32_bits():
    tokens, topk, n = 70000, 8, 4096  # 4.6 GB of rows
    g = torch.Generator(device=DEV).manual_seed(1)
    idx = torch.randperm(tokens * topk, generator=g, device=DEV).to(torch.int32).view(tokens, topk)
    x = torch.randn(tokens, n, generator=g, device=DEV, dtype=torch.float32).to(BF16)
    rows = flux_amd.moe_permute(x, idx)
    probe = torch.randint(0, tokens, (500,), generator=g, device=DEV)
    for j in (0, 7):
        assert torch.equal(rows[idx[probe, j].long()], x[probe])
    w = torch.full((tokens, topk), 0.125, device=DEV)
    assert torch.equal(flux_amd.moe_unpermute(rows, idx, w), x)  # eight eighths of a value are exact
    grad_rows, grad_w = flux_amd.moe_unpermute_backward(x, rows, idx, w)
    assert torch.equal(grad_rows[idx[probe, 3].long()], x[probe] * 0.125)
    square = x[probe].double().square().sum(1)
    assert ((grad_w[probe, 5].double() - square).abs() <= (n / 8 + 16) * 2.0**-24 * square).all()


@pytest.mark.parametrize("topk", [1, 2, 5, 8])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_unpermute_has_the_bits_of_the_gather_reduce(dtype, topk):
    """topk_weighted_gather_reduce, whose weights lie by row: the same multiply-adds in the same order, one rounding (fp32 rows: to bf16)."""
    tokens, n = 333, 1048
    idx, rows = make_index(tokens, topk, 0.2, topk, shuffled=True), data(tokens * topk, n, dtype, 3)
    w = torch.rand(tokens, topk, generator=torch.Generator().manual_seed(topk)).to(DEV)
    by_row = torch.zeros(tokens * topk, device=DEV)
    by_row[idx[idx >= 0].long()] = w[idx >= 0]
    for weights, row_weight in ((w, by_row), (None, None)):
        want = flux_amd.topk_weighted_gather_reduce([rows], idx.flatten(), topk, row_weight)
        assert torch.equal(flux_amd.moe_unpermute(rows, idx, weights).to(want.dtype), want)


@pytest.mark.parametrize("dtype,n", [(BF16, 2047), (F16, 1536), (F32, 7168)])
def test_a_token_has_the_same_sums_in_every_batch(dtype, n):
    """Rows and sums over a token's pairs have the bits of a small batch in a large one, where other forms of the kernels run.  (The weights' gradients need not:
    the lanes that share a token's products are fewer where tokens are many.)"""
    topk, few, many = 3, 40, 20000
    g = torch.Generator(DEV).manual_seed(n)
    idx = torch.randperm(many * topk, generator=g, device=DEV).to(torch.int32).view(many, topk)
    x, rows = (torch.randn(r, n, generator=g, device=DEV).to(dtype) for r in (many, many * topk))
    w = torch.rand(many, topk, generator=g, device=DEV)
    small = torch.arange(few * topk, dtype=torch.int32, device=DEV).view(few, topk)
    small_rows = rows[idx[:few].long().flatten()]
    assert torch.equal(flux_amd.moe_unpermute(small_rows, small, w[:few]), flux_amd.moe_unpermute(rows, idx, w)[:few])
    assert torch.equal(flux_amd.moe_unpermute_backward(x[:few], small_rows, small, w[:few])[0],
                       flux_amd.moe_unpermute_backward(x, rows, idx, w)[0][idx[:few].long().flatten()])


@pytest.mark.parametrize("topk", [1, 2, 4, 6, 8])
@pytest.mark.parametrize("dtype,n", [(BF16, 2047), (F16, 1032), (F32, 1025), (BF16, 45), (F32, 3)])
def test_rows_of_many_megabytes(dtype, n, topk):
    """From 64 MB on the experts' rows pass the caches by: every number of pairs that is requested together, dropped pairs, widths with a rest."""
    print(f"[case] many megabytes {topk} {n} {dtype}", flush=True)
    tokens = (65 << 20) // (topk * n * (4 if dtype == F32 else 2)) + 1
    g = torch.Generator(DEV).manual_seed(n + topk)
    pairs = tokens * topk
    idx = torch.randperm(pairs, generator=g, device=DEV).to(torch.int32).view(tokens, topk)
    idx = torch.where(torch.rand(tokens, topk, generator=g, device=DEV) < 0.1, -1, idx)
    x, rows = (torch.randn(r, n, generator=g, device=DEV).to(dtype) for r in (tokens, pairs))
    w = torch.rand(tokens, topk, generator=g, device=DEV)
    assert torch.equal(capi.moe_permute(x, idx, out=torch.full_like(rows, float("nan"))).double(), want_rows(x, idx))
    out, magnitude = torch.zeros(tokens, n, dtype=torch.float64, device=DEV), torch.zeros(tokens, n, dtype=torch.float64, device=DEV)
    dot, dots = torch.zeros(tokens, topk, dtype=torch.float64, device=DEV), torch.zeros(tokens, topk, dtype=torch.float64, device=DEV)
    for j in range(topk):  # (a column of the index at a time: the terms of all together are gigabytes)
        term = pair_rows(rows, idx[:, j])
        out += term * w[:, j].double()[:, None]
        magnitude += (term * w[:, j].double()[:, None]).abs()
        dot[:, j], dots[:, j] = (term * x.double()).sum(1), (term * x.double()).abs().sum(1)
    close(flux_amd.moe_unpermute(rows, idx, w), out, magnitude, topk + 1)
    grad_rows, grad_w = flux_amd.moe_unpermute_backward(x, rows, idx, w)
    want = want_rows(x, idx, w)
    close(grad_rows, want, want.abs(), 1)
    close(grad_w, dot, dots, n / 8 + 16)


@pytest.mark.parametrize("dtype,n", [(BF16, 1), (F32, 1), (BF16, 3)])
def test_very_many_short_rows(dtype, n):
    """Four bytes a pair for every 65536 rows are more than a row: all rows are cleared before the launch."""
    tokens, topk = 90001, 4
    idx = make_index(tokens, topk, 0.3, 1)
    x = torch.arange(1, tokens * n + 1, device=DEV).remainder(251).add(1).to(dtype).view(tokens, n)
    want = torch.zeros(tokens * topk, n, dtype=dtype, device=DEV)
    live = idx >= 0
    want[idx[live].long()] = x.repeat_interleave(topk, 0).view(tokens, topk, n)[live]
    assert torch.equal(flux_amd.moe_permute(x, idx), want)
    grad_rows, grad_w = flux_amd.moe_unpermute_backward(x, want, idx, torch.full((tokens, topk), 2.0, device=DEV))
    assert torch.equal(grad_rows, want * 2)
    assert torch.equal(grad_w, (x.float() ** 2).sum(1, keepdim=True) * live)


# ---- gradients through autograd ------------------------------------------------------------------------------------


def leaves(tokens=19, topk=3, n=70, seed=3):
    idx = make_index(tokens, topk, 0.2, seed)
    x, w = data(tokens, n, F32, seed), torch.rand(tokens, topk, generator=torch.Generator().manual_seed(seed)).to(DEV)
    return idx, x.requires_grad_(), w.requires_grad_()


def layer(x, idx, w):
    """Tokens to their rows, a stand-in for the experts, and back."""
    return flux_amd.moe_unpermute(torch.tanh(flux_amd.moe_permute(x, idx)), idx, w)


def test_gradients_of_a_run_of_them():
    idx, x, w = leaves()
    out = layer(x, idx, w)
    up = data(*out.shape, F32, 8)
    out.backward(up)
    x64, w64 = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    named = (idx >= 0).double()
    want = ((w64 * named).unsqueeze(-1) * torch.tanh(x64).unsqueeze(1)).sum(1)
    want.backward(up.double())
    assert torch.allclose(out.double(), want, rtol=1e-5, atol=1e-5)
    assert torch.allclose(x.grad.double(), x64.grad, rtol=1e-5, atol=1e-5)
    assert torch.allclose(w.grad.double(), w64.grad, rtol=1e-5, atol=1e-4)
    # against differences, along one direction: central differences of step h are off by h^2 / 6 of a third derivative of order 1, and by
    # roundings of fp32 outputs of order 1 over the step
    dx, dw, h = data(*x.shape, F32, 9), data(*w.shape, F32, 10), 1e-2
    with torch.no_grad():
        f = lambda s: (layer(x + s * dx, idx, w + s * dw).double() * up.double()).sum()  # noqa: E731
        slope = (f(h) - f(-h)) / (2 * h)
    along = (x.grad.double() * dx).sum() + (w.grad.double() * dw).sum()
    scale = (up.abs().double().sum())
    assert (slope - along).abs() <= scale * (10 * h * h + 8 * 2.0**-24 / h)


def test_gradients_that_are_not_wanted_and_broadcast_ones():
    idx, x, w = leaves()
    rows = flux_amd.moe_permute(x.detach(), idx)
    out = flux_amd.moe_unpermute(rows, idx, w)
    out.sum().backward()  # the gradient of a sum is one value with strides of 0
    assert rows.grad is None
    ones = torch.ones_like(out)
    assert torch.equal(w.grad, flux_amd.moe_unpermute_backward(ones, rows, idx, w.detach())[1])
    rows.requires_grad_()
    flux_amd.moe_unpermute(rows, idx, w.detach()).sum().backward()
    assert torch.equal(rows.grad, flux_amd.moe_unpermute_backward(ones, rows.detach(), idx, w.detach())[0])
    rows.grad = None
    flux_amd.moe_unpermute(rows, idx).sum().backward()
    assert torch.equal(rows.grad, flux_amd.moe_permute(ones, idx))
    flux_amd.moe_permute(x, idx).t().contiguous().sum().backward()
    assert torch.equal(x.grad, (idx >= 0).sum(1, keepdim=True).float().expand_as(x))


def test_second_derivatives_are_refused():
    idx, x, w = leaves()
    with pytest.raises(RuntimeError, match="gradient of the gradient"):
        torch.autograd.grad(layer(x, idx, w).sum(), [x, w], create_graph=True)


def test_forward_mode_is_refused():
    """A tangent of the weights, and one that comes with a gradient (forward over reverse), would be lost."""
    ad = torch.autograd.forward_ad
    idx, x, w = leaves()
    rows = flux_amd.moe_permute(x.detach(), idx)
    with ad.dual_level():
        dual_w = ad.make_dual(w.detach(), torch.ones_like(w))
        for call in (lambda: flux_amd.moe_unpermute(rows, idx, dual_w), lambda: flux_amd.moe_unpermute_backward(x.detach(), rows, idx, dual_w)):
            with pytest.raises(RuntimeError, match="weights: forward-mode derivatives"):
                call()
        for out in (flux_amd.moe_permute(x, idx), flux_amd.moe_unpermute(rows.requires_grad_(), idx), flux_amd.moe_unpermute(rows, idx, w)):
            up = ad.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="permute: forward-mode derivatives"):
                out.backward(up)


# ---- streams, graphs, refusals -------------------------------------------------------------------------------------


def test_on_another_stream():
    idx, x = make_index(500, 4, 0.1, 1), data(500, 2048, BF16, 1)
    want = flux_amd.moe_permute(x, idx)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = x * 2
        got = flux_amd.moe_permute(y, idx)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want * 2)


def test_graph_of_a_training_step_replays():
    """Forward and backward in one graph, twice in the same process, with eager work between the replays."""
    tokens, topk, n = 257, 3, 520
    idx, x, w = make_index(tokens, topk, 0.1, 5), data(tokens, n, BF16, 1), torch.rand(tokens, topk, device=DEV)
    up = data(tokens, n, BF16, 2)

    def step():
        rows = flux_amd.moe_permute(x, idx)
        out = flux_amd.moe_unpermute(rows, idx, w)
        grad_rows, grad_w = flux_amd.moe_unpermute_backward(up, rows, idx, w)
        return out, grad_w, flux_amd.moe_permute_backward(grad_rows, idx)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, step()))
        graphs[-1] = (g, graphs[-1][1])
    for seed in range(4):
        x.copy_(data(tokens, n, BF16, 20 + seed))
        idx.copy_(make_index(tokens, topk, 0.1 * seed, 30 + seed))
        want = step()
        for g, got in graphs:
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)


def test_captured_backward_pass():
    """The recorded gradients in a graph; refused while an eager graph of the same leaves is alive, whose stream the capture would draw in."""
    idx, x, w = leaves()

    def step():
        return torch.autograd.grad(layer(x, idx, w).sum(), [x, w])

    alive = flux_amd.moe_permute(x, idx)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
        with torch.cuda.graph(g):
            flux_amd.moe_unpermute(flux_amd.moe_permute(x, idx), idx).sum().backward()
    del alive, g
    x.grad = w.grad = None
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for seed in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, device=DEV, generator=torch.Generator(DEV).manual_seed(seed)))
        want = step()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_lazy_views():
    """What a conjugate view stands for is copied once it is resolved; a negative view of the weights is refused."""
    idx = make_index(30, 2, 0.2, 1)
    x = torch.view_as_complex(torch.randn(30, 17, 2, device=DEV))
    with pytest.raises(RuntimeError, match="conjugate or negative view"):
        flux_amd.moe_permute(x.conj(), idx)
    got = torch.view_as_real(flux_amd.moe_permute(x.conj().resolve_conj(), idx))
    assert torch.equal(got.reshape(60, 34).double(), want_rows(torch.view_as_real(x.conj().resolve_conj()).reshape(30, 34), idx))
    with pytest.raises(RuntimeError, match="weights is a conjugate or negative view"):
        flux_amd.moe_unpermute(data(60, 8, F32, 1), idx, torch._neg_view(torch.ones(30, 2, device=DEV)))
    # a gradient that comes as one
    rows, w = data(60, 8, F32, 1).requires_grad_(), torch.ones(30, 2, device=DEV, requires_grad=True)
    up = torch.ones(30, 8, device=DEV)
    for call, leaf in ((lambda: flux_amd.moe_unpermute(rows, idx), rows), (lambda: flux_amd.moe_unpermute(rows, idx, w), w)):
        want = torch.autograd.grad(call(), leaf, -up)[0]
        assert torch.equal(torch.autograd.grad(call(), leaf, torch._neg_view(up))[0], want)


def test_refusals():
    idx, x, w = make_index(4, 2, 0.0, 1), torch.zeros(4, 16, device=DEV), torch.ones(4, 2, device=DEV)
    rows = torch.zeros(8, 16, device=DEV)
    for call, message in (
        (lambda: flux_amd.moe_permute(x.t(), idx), "contiguous"),
        (lambda: flux_amd.moe_permute(x[0], idx), "2 dimensions"),
        (lambda: flux_amd.moe_permute(x[:3], idx), "tokens"),
        (lambda: flux_amd.moe_permute(x, idx.long()), "Inconsistency"),
        (lambda: flux_amd.moe_permute(x, idx.view(-1)), "2 dimensions"),
        (lambda: flux_amd.moe_permute(x, idx.t()), "contiguous"),
        (lambda: flux_amd.moe_permute(x, idx.cpu()), "device tensor"),
        (lambda: flux_amd.moe_permute_backward(x, idx), "one row per entry"),
        (lambda: flux_amd.moe_permute_backward(rows.double(), idx), "bfloat16, float16 or float32"),
        (lambda: flux_amd.moe_unpermute(rows, idx, w[:, :1]), "weights shape"),
        (lambda: flux_amd.moe_unpermute(rows, idx, w.double()), "bfloat16, float16 or float32"),
        (lambda: flux_amd.moe_unpermute(rows, idx, w.cpu()), "device tensor"),
        (lambda: flux_amd.moe_unpermute(x, idx, w), "one row per entry"),
        (lambda: flux_amd.moe_unpermute_backward(x.half(), rows, idx, w), "grad_out is"),
        (lambda: flux_amd.moe_unpermute_backward(x[:, :8].contiguous(), rows, idx, w), "shape mismatch"),
        (lambda: flux_amd.moe_permute(x, torch.zeros(4, 65, dtype=torch.int32, device=DEV)), "topk=65"),
    ):
        with pytest.raises(RuntimeError, match=message):
            call()
