"""GPU: the routing gradient of softmax scores where one expert has nearly all the weight.

What is left for the gradient there is 1 - s, 1e-5 ... 1e-9; every entry is compared relative to itself and to that share.  The
choices' own terms are in 64 bits and rounded once (2^-24).  Without renormalisation the rest of the row enters through 32-bit
exponentials: 2^-22 each, and 2^-24 of the exponent's size, which is at most 24 here."""
import pytest
import torch

from oracle import posttrain_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("tokens,experts,top_k", [(100, 32, 4), (64, 256, 8), (9000, 64, 6), (50, 500, 16), (40, 2, 2)])
def test_a_dominated_row_keeps_its_digits(cuda, tokens, experts, top_k, renorm):
    from fast_moe_ranking import route_experts

    g = torch.Generator().manual_seed(tokens)
    logits = torch.randn(tokens, experts, generator=g).clamp(-3.0, 3.0) - 14.0
    logits[torch.arange(tokens), torch.randint(0, experts, (tokens,), generator=g)] = torch.rand(tokens, generator=g) * 5
    alpha = 1.0 if renorm else 1.5
    x = logits.to(cuda).requires_grad_(True)
    w, idx = route_experts(x, top_k, renormalize=renorm, scaling_factor=alpha)
    cot = torch.randn(tokens, top_k, generator=g)
    (grad,) = torch.autograd.grad(w, x, cot.to(cuda))
    x64 = logits.double().requires_grad_(True)
    s64 = ref.weights(x64, idx.cpu(), "softmax", renorm, alpha)
    (want,) = torch.autograd.grad(s64, x64, cot.double())
    # in 64 bits the elementary gradient itself is good to 1e-15 of the cotangent
    share = 1.0 - s64.detach()[:, :1] / alpha                    # what the dominant expert leaves to all others
    assert float(share.max()) < 2e-3
    each = 2.0 ** -23 if renorm else 2.0 ** -22 + 2.0 ** -24 * 24 * 2
    size = alpha * cot.double().abs().amax(1, keepdim=True)
    off = (grad.cpu().double() - want).abs()
    bound = each * want.abs() + (0.0 if renorm else each * size * share) + 1e-14 * size
    assert bool((off <= bound).all()), float((off / bound).max())
    # shifting all logits shifts nothing: the row's gradient sums to 0
    total = grad.cpu().double().sum(1).abs()
    assert bool((total <= grad.cpu().double().abs().sum(1) * 4 * each + 1e-13 * size[:, 0]).all())


def test_rows_of_few_and_of_no_experts(cuda):
    """-inf logits among and instead of the choices, for softmax with and without renormalisation."""
    from fast_moe_ranking import route_experts

    for renorm in (True, False):
        x = torch.full((6, 40), float("-inf"))
        x[0, 3] = 1.0
        x[1, [2, 30]] = torch.tensor([0.5, 20.0])
        x[2] = 0.0
        x[3, 1:] = 0.0
        y = x.to(cuda).requires_grad_(True)
        w, idx = route_experts(y, 4, renormalize=renorm)
        cot = torch.randn(6, 4, generator=torch.Generator().manual_seed(1))
        (grad,) = torch.autograd.grad(w, y, cot.to(cuda))
        assert bool(torch.isfinite(grad).all()) and bool((grad.cpu()[torch.isneginf(x)] == 0).all())
        x64 = torch.where(torch.isneginf(x), -800.0, x.double())[:4].requires_grad_(True)
        (want,) = torch.autograd.grad(ref.weights(x64, idx.cpu()[:4], "softmax", renorm, 1.0), x64, cot.double()[:4])
        torch.testing.assert_close(grad.cpu().double()[:4], want, rtol=2.0 ** -21, atol=1e-14)
        assert bool((grad[4:] == 0).all())


def test_weights_are_changed_in_place_like_any_tensor(cuda):
    """Masking or scaling them in place changes nothing that the gradient needs."""
    from b2g import ops
    from fast_moe_ranking import route_experts

    g = torch.Generator(device=cuda).manual_seed(5)
    logits = torch.randn(300, 64, generator=g, device=cuda)
    keep = (torch.rand(300, 6, generator=g, device=cuda) < 0.7).float()
    cot = torch.randn(300, 6, generator=g, device=cuda)
    for fn in ("softmax", "sigmoid", "sqrtsoftplus"):
        for renorm in (True, False):
            x = logits.clone().requires_grad_(True)
            w, idx = route_experts(x, 6, score_function=fn, renormalize=renorm)
            (want,) = torch.autograd.grad(w * keep, x, cot)
            w, _ = route_experts(x, 6, score_function=fn, renormalize=renorm)
            w.mul_(keep)
            (got,) = torch.autograd.grad(w, x, cot)
            assert torch.equal(got, want)
            assert torch.equal(ops.route_experts_bwd(cot * keep, logits, None, idx, fn, renorm), want)
            assert torch.equal(ops.route_experts_bwd(cot * keep, logits, w.detach(), idx, fn, renorm), want)
    with pytest.raises(TypeError, match="grad_weights"):
        ops.route_experts_bwd(None, logits, None, idx)
