"""GPU: the preference loss where several CTAs share a pair, with sequences whose lengths have nothing to do with one another.

Long sequences on average give every pair a cluster, whose CTAs send their sums to the first one's shared memory.  CTAs without
tokens of their own come to that at once, those of a long sequence much later.  Sums are in 64 bits, results rounded to 32 once, beta
is rounded to 32: 2^-22 relative, and 1e-14 of the sum of all magnitudes."""
import pytest
import torch

from oracle import posttrain_ref as ref

pytestmark = pytest.mark.gpu


def _case(lengths, seed, behind=0):
    g = torch.Generator().manual_seed(seed)
    ends = torch.tensor([0] + list(lengths)).cumsum(0)
    n = int(ends[-1]) + behind
    logp = -torch.rand(n, generator=g, dtype=torch.float64) * 1e-3
    rf = (logp + 1e-4 * torch.randn(n, generator=g, dtype=torch.float64)).float()
    target = torch.where(torch.rand(n, generator=g) < 0.2, -100, 1)
    return logp, rf, target, ends


@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("lengths,behind", [
    ([0, 70000], 0), ([70000, 0], 0), ([0, 0], 60000),                              # nothing on one side, nothing at all in a long buffer
    ([1, 0, 2, 0, 120000, 0, 3, 0], 0), ([0, 5, 0, 1, 0, 0, 90001, 1], 0),          # short pairs beside a long sequence
    ([3000, 1, 2999, 40001, 0, 7, 2049, 2048], 100000)])                            # a buffer longer than its answers
def test_pairs_of_unequal_lengths(cuda, lengths, behind, average):
    from b2g import autograd as ag

    logp, rf, target, ends = _case(lengths, len(lengths) + behind, behind)
    assert len(logp) // len(lengths) > 2048                                         # more than one CTA a pair
    x64 = logp.clone().requires_grad_(True)
    want = ref.preference(x64, ends, rf, 0.1, 0.0, "sigmoid", average, target)
    x = logp.to(cuda).requires_grad_(True)
    on = (x, ends.to(cuda), rf.to(cuda), 0.1, 0.0, "sigmoid", average, target.to(cuda))
    first = ag.preference_loss(*on)
    slack = float(logp.abs().sum() + rf.double().abs().sum()) * 1e-14
    for a, b in zip(first, want):
        torch.testing.assert_close(a.detach().cpu().double(), b.detach(), rtol=2.0 ** -22, atol=slack)
    (grad,) = torch.autograd.grad(first[0].sum(), x)
    (want_grad,) = torch.autograd.grad(want[0].sum(), x64)
    torch.testing.assert_close(grad.cpu(), want_grad, rtol=2.0 ** -21, atol=0)
    for _ in range(20):                                                             # launches straight behind one another
        again = ag.preference_loss(*on)
        assert all(torch.equal(a, b) for a, b in zip(again, first))
