"""GPU: digits of the row losses where something cancels: 1 - p of a nearly certain target, temperatures, sums of many terms."""
import math

import pytest
import torch

from oracle import posttrain_ref as ref

pytestmark = pytest.mark.gpu


def _confident(rows, vocab, seed):
    """fp32 rows whose target has all but 1e-5 ... 1e-9 of the probability."""
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(rows, vocab, generator=g)
    target = torch.randint(0, vocab, (rows,), generator=g)
    target[0], target[1] = 0, vocab - 1
    rest = torch.linspace(math.log(1e-5), math.log(1e-9), rows)
    logits[torch.arange(rows), target] = (torch.logsumexp(logits.double(), 1) - rest.double()).float()
    return logits, target


@pytest.mark.parametrize("tau", [1.0, 0.8])
@pytest.mark.parametrize("rows,vocab", [(16, 2), (16, 300), (16, 3001), (16, 9001), (40, 32003), (12, 131071), (4, 500001)])
def test_the_entry_of_a_nearly_certain_target_in_fp32(cuda, rows, vocab, tau):
    """It is coef (1 - p)/tau, and 1 - p is the sum of the other exponentials over all of them: 2^-22 of each exponential, 2^-23 of
    its exponent's size (difference and scaling half a step each; at most 40 here), 2^-22 for the four factors.  The sum over the row is
    0 but for those factors and half a step of every entry."""
    from b2g import ops

    logits, target = _confident(rows, vocab, vocab)
    logits = logits * tau
    x, t = logits.to(cuda), target.to(cuda)
    p = torch.softmax(logits.double() / tau, 1)
    at = (torch.arange(rows), target)
    rest = p.clone()
    rest[at] = 0.0
    rest = rest.sum(1)
    assert float(rest.max()) < 1e-4 and float(rest.min()) < 1e-8
    adv = torch.linspace(0.5, -1.5, rows) + 0.01
    coef = -adv.double() / tau                                       # old_logp is None: the ratio is 1
    grad = ops.policy_loss(x, t, adv.to(cuda), temperature=tau)[3]
    _, stats = ops.token_logprobs(x, t, tau)
    back = ops.token_logprobs_bwd(-adv.to(cuda), x, t, stats, tau)
    each = 2.0 ** -21 + 40 * 2.0 ** -23
    for got in (grad.cpu().double(), back.cpu().double()):
        off = (got[at] - coef * rest).abs() / (coef * rest).abs()
        assert bool((off <= each).all()), float(off.max())
        total, size = got.sum(1).abs(), got.abs().sum(1)
        assert bool((total <= size * 2.0 ** -20).all()), float((total / size).max())


def test_a_shift_of_all_logits_changes_no_gradient(cuda):
    """Shifts that leave the differences of the logits as they are (logits on a grid of 2^-6, shifted by up to 20480)."""
    from b2g import ops

    g = torch.Generator().manual_seed(3)
    for vocab in (300, 9001, 32003):
        logits = torch.round(torch.randn(8, vocab, generator=g) * 64) / 64
        target = torch.randint(0, vocab, (8,), generator=g)
        logits[torch.arange(8), target] = 16.0 + torch.arange(8).float()
        adv = torch.ones(8, device=cuda)
        want = ops.policy_loss(logits.to(cuda), target.to(cuda), adv)[3]
        for shift in (64.0, -1024.0, 8192.0, 20480.0):
            got = ops.policy_loss((logits + shift).to(cuda), target.to(cuda), adv)[3]
            assert torch.equal((logits + shift) - shift, logits)
            torch.testing.assert_close(got, want, rtol=2.0 ** -20, atol=0)
