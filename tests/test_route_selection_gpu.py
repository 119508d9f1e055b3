"""GPU: the choice of experts equals the order of the choices in 64 bits, where 32 bits put experts, or groups, in another one.

Every comparison of ids is exact; the oracle sorts in Python's floats."""
import pytest
import torch

from oracle import posttrain_ref as ref

pytestmark = pytest.mark.gpu

SCORES = ("softmax", "sigmoid", "sqrtsoftplus")


def _same(cuda, logits, bias, fn, top_k, groups=1, kept=1, best=1):
    from b2g import ops

    _, idx = ops.route_experts(logits.to(cuda), top_k, bias.to(cuda), fn, groups, kept, best)
    want = ref.choose(logits, top_k, bias, fn, groups, kept, best)
    wrong = (idx.cpu() != want).any(1)
    assert not bool(wrong.any()), (fn, int(wrong.sum()), idx.cpu()[wrong][:2].tolist(), want[wrong][:2].tolist())


@pytest.mark.parametrize("experts", [8, 32, 40, 256])
def test_a_large_score_under_a_large_negative_bias(cuda, experts):
    """The first two choices are 1.2e-8 apart, which is clear of their own errors; the third expert's is a difference of two
    numbers near 1, stands behind both in 32 bits and before them in 64."""
    logits = torch.full((1, experts), -20.0)
    bias = torch.full((experts,), -1.0)
    logits[0, 2] = 2.89365625
    bias[:3] = torch.tensor([0.01, 0.0099999877, -0.93753195])
    _same(cuda, logits, bias, "sigmoid", 1)
    # as many such rows as there are places for the expert, and steps of its bias around the border
    rows = torch.full((32, experts), -20.0)
    for step in range(-4, 5):
        b = torch.full((experts,), -1.0)
        b[0], b[1] = 0.01, 0.0099999877
        b[7] = -0.93753195 + step * 2.0 ** -24
        rows[:, 7] = 2.89365625 + (torch.arange(32) - 16) * 2.0 ** -22
        for top_k in (1, 2, 3):
            _same(cuda, rows, b, "sigmoid", top_k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_experts_at_the_border(cuda, dtype):
    """Same logit and same bias: equal by construction, and no reason not to look at who comes next."""
    logits = torch.full((4, 24), -20.0)
    logits[0, :3] = torch.tensor([18.0, 18.0, 18.125])
    logits[1, [4, 9, 20]] = torch.tensor([18.0, 18.0, 18.125])
    logits[2, :6] = torch.tensor([18.0, 18.0, 18.0, 18.0, 18.0, 18.125])
    logits[3, 10:16] = torch.tensor([18.125, 18.0, 18.0, 18.25, 18.0, 18.0])
    for top_k in (1, 2, 3, 5):
        _same(cuda, logits.to(dtype), torch.zeros(24), "sigmoid", top_k)
    # a softmax tail of duplicated logits under one dominant logit: every tail choice is the bias in 32 bits
    g = torch.Generator().manual_seed(1)
    for experts in (20, 48, 64):
        tail = (torch.randint(-8, 8, (200, experts), generator=g) * 0.125)
        tail[:, 5] = 40.0
        for top_k in (1, 2, 3, 8):
            _same(cuda, tail.to(dtype), torch.full((experts,), 0.25), "softmax", top_k)


@pytest.mark.parametrize("fn", SCORES)
@pytest.mark.parametrize("experts", [6, 32, 64, 130])
def test_choices_brought_together_by_their_biases(cuda, fn, experts):
    """Scores of all sizes whose choices lie within some 1e-7 of one another, a third of them duplicated."""
    g = torch.Generator().manual_seed(experts)
    spread = {"softmax": 3.0, "sigmoid": 6.0, "sqrtsoftplus": 40.0}[fn]
    for trial in range(6):
        base = (torch.rand(experts, generator=g) - 0.5) * 2 * spread
        half = max(1, experts // 6)
        base[half:2 * half] = base[:half]
        s = ref.scores(base[None].double(), fn)[0]
        bias = (0.3 - s + torch.randn(experts, generator=g, dtype=torch.float64) * 2e-7).float()
        bias[half:2 * half] = bias[:half]
        logits = base[None] * (1 + torch.randn(64, 1, generator=g) * 2e-7)      # an equal factor keeps duplicates equal
        for top_k in (1, 2, min(6, experts - 1)):
            _same(cuda, logits, bias, fn, top_k)


@pytest.mark.parametrize("experts,groups,best", [(16, 8, 2), (64, 32, 2), (128, 16, 2), (24, 4, 1), (96, 8, 2)])
def test_groups_whose_two_best_cancel(cuda, experts, groups, best):
    """A choice near +64 and one near -64: what their sum loses in 32 bits is a step of 64, whatever the sum's own size is."""
    g = torch.Generator().manual_seed(experts)
    per = experts // groups
    for fn in SCORES:
        bias = torch.full((groups, per), -200.0)
        bias[:, 0], bias[:, 1] = 64.0, -64.0
        logits = torch.randn(200, experts, generator=g) * (1e-5 * experts if fn == "softmax" else 2e-5)
        for kept in (1, groups // 2, groups - 1):
            _same(cuda, logits, bias.reshape(-1), fn, 2, groups, kept, best)


def test_a_group_with_an_undefined_choice_comes_last(cuda):
    from b2g import ops

    for experts, groups in ((8, 4), (64, 4), (256, 8)):
        for fn in SCORES:
            logits = torch.randn(50, experts, generator=torch.Generator().manual_seed(experts))
            bias = torch.zeros(experts)
            bias[1] = float("nan")
            logits[:, :2] = 6.0                       # the best logits are in the group that the NaN spoils
            _, idx = ops.route_experts(logits.to(cuda), 2, bias.to(cuda), fn, groups, groups - 1, 2)
            assert bool((idx >= experts // groups).all()), (experts, fn)
            # with all groups kept it is the expert that comes last, and experts are still distinct
            _, idx = ops.route_experts(logits[:, :8].contiguous().to(cuda), 8, bias[:8].to(cuda), fn, 1, 1, 2)
            assert bool((idx[:, -1] == 1).all()) and bool((idx.sort(1).values.cpu() == torch.arange(8)).all())


def test_experts_taken_out_by_an_infinite_bias(cuda):
    g = torch.Generator().manual_seed(4)
    for fn in SCORES:
        for experts, groups, kept in ((64, 8, 3), (40, 1, 1), (256, 8, 4)):
            logits = torch.randn(64, experts, generator=g)
            bias = torch.randn(experts, generator=g) * 0.1
            bias[::3] = float("-inf")
            _same(cuda, logits, bias, fn, 6, groups, kept, 2)


def test_rows_without_any_expert_are_ordered_by_their_biases(cuda):
    """All logits -inf: every score is 0, and the choices are the biases, however close they lie."""
    for experts, groups, kept in ((16, 1, 1), (40, 1, 1), (64, 8, 4), (256, 8, 3)):
        logits = torch.full((20, experts), float("-inf"))
        bias = 0.5 + torch.randint(-3, 4, (experts,), generator=torch.Generator().manual_seed(experts)) * 2.0 ** -24
        for fn in SCORES:
            _same(cuda, logits, bias, fn, 6, groups, kept, 2)
