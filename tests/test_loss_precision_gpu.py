"""GPU: digits of the row losses where something cancels: 1 - p of a nearly certain target, temperatures, sums of many terms; NaN that
must not get lost."""
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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(256, 3001), (128, 9001), (96, 32003), (64, 129280)])
@pytest.mark.parametrize("tau", [1.0, 0.973, 0.899])
def test_log_probabilities_of_flat_rows(cuda, dtype, rows, vocab, tau):
    """fp64 log-probabilities of rows without a standing-out token, root mean square over the rows.

    A term is off by up to 2^-22 (exponential), 3 * 2^-24 (tree) and 2 * 2^-24 of its exponent, 16 at most for the terms that count;
    uniformly distributed that is 1 / sqrt(3) of it, and the terms' errors are independent: with n = (sum p)^2 / sum p^2 of them
    the sum's is 1 / sqrt(n) of one.  ex2.approx is short by 3.7e-8 ... 5.9e-8 according to the fraction, 4.9e-8 of which is
    put back: 1.2e-8 may be left."""
    from b2g import ops

    g = torch.Generator().manual_seed(vocab + rows)
    logits = (torch.randn(rows, vocab, generator=g) * 1.5).to(dtype)
    target = torch.randint(0, vocab, (rows,), generator=g)
    t32 = float(torch.tensor(tau, dtype=torch.float32))
    want = ref.logprobs(logits.double(), target, t32)
    got = ops.token_logprobs(logits.to(cuda), target.to(cuda), tau, dtype=torch.float64)[0].cpu()
    p = torch.softmax(logits.double() / t32, 1)
    n = 1.0 / (p * p).sum(1)
    one = (2.0 ** -22 + 2.0 ** -24 * (3 + 2 * 16)) / math.sqrt(3.0)
    bound = float((one * one / n).mean().sqrt()) + 1.2e-8
    rms = float((got - want).pow(2).mean().sqrt())
    bias = float((got - want).mean())
    assert rms <= bound, (rms, bias, bound)


def test_equal_logits_show_the_whole_correction(cuda):
    """exp2(0) is exact, and so is what a row of equal logits sums: there the average that is put back for ex2.approx is an error,
    4.9e-8 in every log-probability of bf16 rows.  fp32 rows use no such correction: a double's steps, and 2^-24 of the sum's."""
    from b2g import ops

    for vocab in (1000, 9001, 129280):
        t = torch.tensor([5], device=cuda)
        for dtype, bound in ((torch.bfloat16, 5e-8), (torch.float32, 2.0 ** -30)):
            got = float(ops.token_logprobs(torch.full((1, vocab), 2.5, dtype=dtype, device=cuda), t, dtype=torch.float64)[0])
            assert abs(got + math.log(vocab)) <= bound + 1e-14 * math.log(vocab), (vocab, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [200, 9001, 40003, 1_000_003])
def test_an_undefined_advantage_reaches_the_gradient(cuda, dtype, vocab):
    from b2g import ops

    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn(3, vocab, generator=g).to(dtype).to(cuda)
    target = torch.tensor([1, 2, 3], device=cuda)
    adv = torch.tensor([1.0, float("nan"), -1.0], device=cuda)
    for old in (None, torch.zeros(3, device=cuda)):
        loss, _, _, grad = ops.policy_loss(logits, target, adv, old_logp=old)
        assert bool(torch.isnan(loss[1])) and bool(torch.isnan(grad[1]).all())
        assert bool(torch.isfinite(grad[[0, 2]]).all()) and bool(torch.isfinite(loss[[0, 2]]).all())
