"""GPU: expert routing with groups, balance bias and renormalised weights, and its gradient, against the 64-bit oracle.

Ids are compared exactly.  Weights: exponential, sum, division and scaling in 32 bits at worst, (8 + top_k + spread) half
steps of fp32, the spread being what the exponent's own rounding can be worth.  Gradients: the same again for the factors
in front of the score's slope, relative to the largest entry of the row, plus half a step of the logits' type.
"""
import pytest
import torch

from oracle import posttrain_ref as ref

pytestmark = pytest.mark.gpu


def _route(logits, top_k, **kw):
    from fast_moe_ranking import route_experts

    return route_experts(logits, top_k, **kw)


def _check(cuda, logits, top_k, bias=None, fn="softmax", groups=1, kept=1, best=1, renorm=True, alpha=1.0, seed=0):
    x = logits.to(cuda).requires_grad_(True)
    w, idx = _route(x, top_k, correction_bias=None if bias is None else bias.to(cuda), score_function=fn, num_groups=groups, top_groups=kept,
                    group_experts=best, renormalize=renorm, scaling_factor=alpha)
    assert w.dtype == torch.float32 and idx.dtype == torch.int64 and tuple(idx.shape) == (logits.shape[0], top_k)
    want = ref.choose(logits, top_k, bias, fn, groups, kept, best)
    assert torch.equal(idx.cpu(), want)
    x64 = logits.double().requires_grad_(True)
    w64 = ref.weights(x64, want, fn, renorm, alpha)
    finite = logits.double().masked_fill(torch.isneginf(logits.double()), 0.0)
    tol = (8 + top_k + float(finite.abs().max()) * 2) * 2.0 ** -24
    torch.testing.assert_close(w.detach().cpu().double(), w64.detach(), rtol=tol, atol=1e-37)
    g = torch.randn(w.shape, generator=torch.Generator().manual_seed(seed))
    (grad,) = torch.autograd.grad(w, x, g.to(cuda))
    (want_grad,) = torch.autograd.grad(w64, x64, g.double())
    want_grad = torch.where(torch.isneginf(x64.detach()), torch.zeros_like(want_grad), want_grad)   # autograd's 0 * inf
    assert grad.dtype == logits.dtype
    scale = (g.double().abs() * w64.detach()).sum(1, keepdim=True) + g.double().abs().amax(1, keepdim=True) * w64.detach().amax(1, keepdim=True)
    off = (grad.cpu().double() - want_grad).abs()
    assert bool((off <= want_grad.abs() * ref.HALF[logits.dtype] + 2 * tol * scale + 1e-37).all()), float((off / scale).max())


@pytest.mark.parametrize("fn", ["softmax", "sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,experts,top_k,groups,kept,best", [
    (1, 1, 1, 1, 1, 1), (3, 2, 2, 1, 1, 1), (5, 7, 3, 1, 1, 1), (33, 32, 32, 1, 1, 1), (9, 33, 5, 1, 1, 1), (130, 64, 6, 8, 3, 2),
    (21, 96, 5, 4, 2, 1), (7, 100, 9, 10, 4, 2), (257, 256, 8, 8, 4, 2), (11, 257, 4, 1, 1, 1), (17, 512, 16, 32, 2, 2), (6, 384, 8, 32, 5, 1),
    (4, 32, 4, 32, 7, 2), (5, 500, 10, 20, 3, 2)])
def test_against_the_oracle(cuda, fn, renorm, dtype, tokens, experts, top_k, groups, kept, best):
    g = torch.Generator().manual_seed(tokens * 1000 + experts)
    logits = (torch.randn(tokens, experts, generator=g) * 2).to(dtype)
    for bias in (None, torch.randn(experts, generator=g) * 0.1):
        _check(cuda, logits, top_k, bias, fn, groups, kept, best, renorm, 2.5 if renorm else 1.0, seed=experts)


def test_ties_go_to_the_lower_id_and_the_lower_group(cuda):
    for dtype in (torch.bfloat16, torch.float32):
        for fn in ("softmax", "sigmoid", "sqrtsoftplus"):
            flat = torch.zeros(3, 256, dtype=dtype)
            flat[1, 200] = -0.0
            _check(cuda, flat, 8, torch.zeros(256), fn, 8, 4, 2)
            _check(cuda, flat, 8, None, fn, 8, 4, 2)
    # a coarse grid of logits and biases: many equal choices, the tied ones in several lanes
    g = torch.Generator().manual_seed(5)
    logits = torch.randint(-2, 3, (300, 160), generator=g).float()
    bias = torch.randint(0, 2, (160,), generator=g).float() * 0.25
    for fn in ("softmax", "sigmoid", "sqrtsoftplus"):
        _check(cuda, logits, 12, bias, fn, 10, 3, 2)
        _check(cuda, logits.bfloat16(), 12, bias, fn)


def test_choices_that_32_bits_cannot_tell_apart(cuda):
    """Scores that differ by far less than fp32 resolves: saturated sigmoids and softmax tails under one bias, and choices that
    bias and score bring together to within 1e-9."""
    g = torch.Generator().manual_seed(6)
    logits = 17.0 + torch.rand(400, 96, generator=g) * 4          # sigmoid is 1 - 1e-8 ... 1 - 1e-9
    _check(cuda, logits, 8, torch.zeros(96), "sigmoid")
    _check(cuda, -logits, 8, torch.full((96,), 0.5), "sigmoid")    # scores of 1e-8 vanish in the sum with the bias in 32 bits
    base = torch.randn(1, 64, generator=g).double()
    bias = (0.7 - torch.sigmoid(base[0])).float()                  # every choice is 0.7 to within the bias' rounding
    _check(cuda, base.float().expand(5, 64).contiguous(), 8, bias, "sigmoid", 8, 3, 2)
    tail = torch.randn(200, 256, generator=g)
    tail[:, 0] = 60.0                                              # all other probabilities are below 1e-24
    _check(cuda, tail, 8, torch.full((256,), 0.125), "softmax")
    _check(cuda, tail.bfloat16(), 8, torch.full((256,), 0.125), "softmax", 8, 4, 2)


@pytest.mark.parametrize("fn", ["softmax", "sigmoid", "sqrtsoftplus"])
def test_masked_experts_and_extreme_logits(cuda, fn):
    g = torch.Generator().manual_seed(7)
    logits = torch.randn(40, 48, generator=g)
    logits[:, ::3] = float("-inf")
    logits[5:10, 1:] = float("-inf")                               # fewer experts left than are asked for
    _check(cuda, logits[:5], 6, torch.randn(48, generator=g) * 0.1, fn, 4, 2, 2)
    x = logits.to(cuda).requires_grad_(True)
    w, idx = _route(x, 6, score_function=fn)
    assert torch.equal(idx.cpu(), ref.choose(logits, 6, None, fn))
    assert bool((w[5:10, 1:] == 0).all()) and bool(torch.isfinite(w).all())
    (grad,) = torch.autograd.grad(w.sum(), x)
    assert bool(torch.isfinite(grad).all()) and bool((grad[torch.isneginf(logits).to(cuda)] == 0).all())
    # a row without any expert left: ids in order, no weight, no gradient
    for renorm in (True, False):
        y = torch.full((3, 48), float("-inf"), device=cuda, requires_grad=True)
        w, idx = _route(y, 4, score_function=fn, renormalize=renorm)
        assert idx.tolist() == [[0, 1, 2, 3]] * 3 and bool((w == 0).all())
        assert bool((torch.autograd.grad(w, y, torch.ones_like(w))[0] == 0).all())
    big = torch.tensor([[80.0, -80.0, 30.0, -30.0, 0.0, 1e-3, -1e-3, 5.0]])
    _check(cuda, big, 3, None, fn)
    _check(cuda, big, 8, None, fn)
    lowest = torch.full((2, 40), torch.finfo(torch.float32).min)
    w, idx = _route(lowest.to(cuda), 5, score_function=fn)
    assert idx.tolist() == [[0, 1, 2, 3, 4]] * 2 and bool(torch.isfinite(w).all())


def test_nan_and_inf_rows_still_give_distinct_ids(cuda):
    g = torch.Generator().manual_seed(8)
    for fn in ("softmax", "sigmoid", "sqrtsoftplus"):
        for bias in (None, torch.randn(70, generator=g)):
            logits = torch.randn(6, 70, generator=g)
            logits[0] = float("nan")
            logits[1, 3] = float("nan")
            logits[2, 5:9] = float("inf")
            logits[3, ::2] = float("nan")
            b = None if bias is None else bias.to(cuda)
            _, idx = _route(logits.to(cuda), 9, correction_bias=b, score_function=fn, num_groups=7, top_groups=3)
            for row in idx.tolist():
                assert len(set(row)) == 9 and all(0 <= i < 70 for i in row)
            if bias is None and fn != "softmax":
                _, idx = _route(logits.to(cuda), 9, score_function=fn)
                assert 3 not in idx[1].tolist()                    # NaN is chosen last


def test_strided_rows_and_gradients_of_any_layout(cuda):
    g = torch.Generator().manual_seed(9)
    wide = torch.randn(50, 300, generator=g)
    for dtype in (torch.float32, torch.bfloat16):
        for first in (0, 3, 8):
            view = wide.to(dtype).to(cuda)[:, first:first + 256]
            w, idx = _route(view, 8)
            w2, idx2 = _route(view.contiguous(), 8)
            assert torch.equal(w, w2) and torch.equal(idx, idx2)
    x = wide[:, :256].contiguous().to(cuda).requires_grad_(True)
    w, _ = _route(x, 8, score_function="sigmoid", renormalize=False)
    (a,) = torch.autograd.grad(w.sum(), x, retain_graph=True)      # an expanded gradient
    (b,) = torch.autograd.grad(w, x, torch.ones_like(w))
    assert torch.equal(a, b)
    col = torch.randn(8, 50, generator=g).to(cuda).t()
    (c,) = torch.autograd.grad(_route(x, 8)[0], x, col)
    (d,) = torch.autograd.grad(_route(x, 8)[0], x, col.contiguous())
    assert torch.equal(c, d)


def test_gradient_against_differences(cuda):
    """Central differences of the kernel's own weights.  h = 2^-7 keeps every choice (the logits of a row lie 0.05 apart); the
    weights' third derivative is at most 1 times alpha, so truncation is below alpha h^2 = 1.6e-4, and 2^-20 of rounding over 2h
    is below 1.3e-4."""
    g = torch.Generator().manual_seed(10)
    e, k, alpha = 24, 5, 1.5
    logits = torch.stack([torch.randperm(e, generator=g) for _ in range(6)]).float() * 0.05 - 0.5
    cot = torch.randn(6, k, generator=g).to(cuda)
    h = 2.0 ** -7
    for fn in ("softmax", "sigmoid", "sqrtsoftplus"):
        for renorm in (True, False):
            kw = dict(score_function=fn, renormalize=renorm, scaling_factor=alpha)
            x = logits.to(cuda).requires_grad_(True)
            (grad,) = torch.autograd.grad(_route(x, k, **kw)[0], x, cot)
            for col in range(e):
                step = torch.zeros_like(x)
                step[:, col] = h
                with torch.no_grad():
                    (up, iu), (down, id_) = _route(x + step, k, **kw), _route(x - step, k, **kw)
                assert torch.equal(iu, id_)
                diff = ((up - down).double() * cot.double()).sum(1) / (2 * h)
                bound = 3e-4 * cot.abs().sum(1).double()
                assert bool(((diff - grad[:, col].double()).abs() <= bound).all()), (fn, renorm, col)


def test_no_tokens_and_more_tokens_than_one_grid_row(cuda):
    w, idx = _route(torch.zeros(0, 64, device=cuda), 4)
    assert tuple(w.shape) == tuple(idx.shape) == (0, 4)
    x = torch.zeros(0, 64, device=cuda, requires_grad=True)
    assert torch.autograd.grad(_route(x, 4)[0].sum(), x)[0].shape == (0, 64)
    g = torch.Generator(device=cuda).manual_seed(11)
    logits = torch.randn(300_001, 64, generator=g, device=cuda)
    w, idx = _route(logits, 6)
    rows = torch.tensor([0, 65_535, 65_536, 262_144, 300_000])
    assert torch.equal(idx[rows.to(cuda)].cpu(), ref.choose(logits[rows.to(cuda)].cpu(), 6))


def test_streams_and_captured_graph(cuda):
    from b2g import ops

    g = torch.Generator(device=cuda).manual_seed(12)
    logits = torch.randn(512, 256, generator=g, device=cuda)
    bias = torch.randn(256, generator=g, device=cuda) * 0.1
    cot = torch.randn(512, 8, generator=g, device=cuda)

    def both():
        w, idx = ops.route_experts(logits, 8, bias, "sigmoid", 8, 4, 2, True, 2.5)
        return w, idx, ops.route_experts_bwd(cot, logits, w, idx, "sigmoid", True, 2.5)

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    logits.copy_(torch.randn(512, 256, generator=g, device=cuda))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, both()))


def test_refusals(cuda):
    from b2g import ops

    x = torch.zeros(4, 64, device=cuda)
    with pytest.raises(RuntimeError, match="CUDA BF16 or FP32"):
        _route(x.half(), 4)
    with pytest.raises(RuntimeError, match="stride"):
        _route(torch.zeros(64, 4, device=cuda).t(), 4)
    with pytest.raises(RuntimeError, match="overlap"):
        _route(torch.zeros(1, 64, device=cuda).expand(4, 64), 4)
    with pytest.raises(TypeError, match="bias must be"):
        _route(x, 4, correction_bias=torch.zeros(64, device=cuda, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="scaling_factor"):
        _route(x, 4, scaling_factor=0.0)
    w, idx = _route(x, 4)
    with pytest.raises(ValueError, match="grad_weights"):
        ops.route_experts_bwd(torch.zeros(4, 5, device=cuda), x, w, idx)
    y = x.clone().requires_grad_(True)
    (first,) = torch.autograd.grad(_route(y, 4)[0].sum(), y, create_graph=False)
    with pytest.raises(RuntimeError, match="higher-order"):
        torch.autograd.grad(_route(y, 4)[0].sum(), y, create_graph=True)


@pytest.mark.parametrize("fn", ["softmax", "sigmoid", "sqrtsoftplus"])
def test_a_single_renormalised_choice_has_no_gradient(cuda, fn):
    """Its weight is the scaling factor whatever its score is; what is left of the gradient is below 1e-16 of the cotangent."""
    g = torch.Generator().manual_seed(13)
    for dtype in (torch.bfloat16, torch.float32):
        for alpha in (1.0, 1.5, 2.7):
            x = (torch.randn(200, 24, generator=g) * 2).to(dtype).to(cuda).requires_grad_(True)
            w, _ = _route(x, 1, score_function=fn, scaling_factor=alpha)
            assert bool((w == torch.tensor(alpha)).all())
            cot = torch.randn(200, 1, generator=g).to(cuda)
            (grad,) = torch.autograd.grad(w, x, cot)
            assert float(grad.float().abs().max()) < 1e-15 * float(cot.abs().max())


def test_gradient_where_one_expert_has_nearly_all_the_weight(cuda):
    """fp32 logits, a row dominated by one of its choices: 1 - w is 1e-5 ... 1e-9 there, and the gradient is proportional to it.
    Softmax takes it from fp32 weights (off by half a step of 1), the other scores from the logits in 64 bits."""
    g = torch.Generator().manual_seed(14)
    logits = torch.randn(100, 32, generator=g) - 14.0
    logits[:, 3] = 2.0
    for fn, tol in (("sigmoid", 2.0 ** -22), ("sqrtsoftplus", 2.0 ** -22)):
        x = logits.to(cuda).requires_grad_(True)
        w, idx = _route(x, 4, score_function=fn)
        cot = torch.randn(100, 4, generator=g)
        (grad,) = torch.autograd.grad(w, x, cot.to(cuda))
        x64 = logits.double().requires_grad_(True)
        (want,) = torch.autograd.grad(ref.weights(x64, idx.cpu(), fn, True, 1.0), x64, cot.double())
        off = (grad.cpu().double() - want).abs()
        scale = want.abs().amax(1, keepdim=True)
        assert bool((off <= tol * want.abs() + 2.0 ** -40 * scale).all()), fn
