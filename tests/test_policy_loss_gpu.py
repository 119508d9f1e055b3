"""GPU: token log-probabilities, the clipped policy loss and the preference loss against the 64-bit oracle.

Tolerances.  A log-probability is off by ``oracle.posttrain_ref.lse_error`` (the 32-bit exponentials) plus half a step of its
type.  A cotangent entry c (onehot - p): the factor c is off by what the log-probability's error makes of the ratio and the KL
term; p by that error and by 2^-22 + 2^-23 |t| of its own exponential (|t| the exponent's size); at the target 1 - p keeps
p's absolute error and, for fp32 logits, half a step of z/tau, m/tau and lse each; then half a step of the type.
"""
import ctypes as C
import math

import pytest
import torch

from oracle import posttrain_ref as ref

pytestmark = pytest.mark.gpu


def _rows(n, vocab, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(n, vocab, generator=g) * spread
    target = torch.randint(0, vocab, (n,), generator=g)
    logits[torch.arange(n), target] += 3.0 + 6.0 * torch.rand(n, generator=g)
    return logits.to(dtype), target


def _logp_tol(logp, vocab, dtype=torch.float32):
    return ref.lse_error(vocab) + (logp.abs() * 2.0 ** -24 if dtype == torch.float32 else 0.0)


def _check_cotangent(got, logits, target, coef, coef_tol, tau, dtype, live):
    """got vs coef (onehot - softmax)/tau with the bounds of the module's text."""
    n, v = logits.shape
    z = logits.double() / tau
    z = torch.where(live[:, None], z, torch.zeros_like(z))
    lse = torch.logsumexp(z, 1, keepdim=True)
    p = torch.softmax(z, 1)
    want = -p.clone()
    hot = torch.arange(n), target.clamp(min=0)
    want[hot] += 1.0
    c = (torch.where(live, coef, torch.zeros_like(coef)) / tau)[:, None]
    t = (z.amax(1, keepdim=True) - z).clamp(max=200.0)
    p_tol = p * (ref.lse_error(v) + 2.0 ** -22 + 2.0 ** -23 * t + 2.0 ** -22)
    if dtype == torch.float32:
        extra = torch.zeros_like(p)
        extra[hot] = 2.0 ** -24 * (z[hot].abs() + z.abs().amax(1) + lse[:, 0].abs()) + 2.0 ** -22
        p_tol = p_tol + extra
    else:
        p_tol[hot] += ref.lse_error(v) + 2.0 ** -24
    bound = (c * want).abs() * ref.HALF[dtype] * 1.01 + c.abs() * p_tol * 1.01 + want.abs() * (coef_tol / tau)[:, None] + 2e-38
    off = (got.cpu().double() - c * want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
    assert bool((got.cpu()[~live] == 0).all())


SHAPES = [(1, 1), (2, 2), (3, 7), (5, 37), (4, 1000), (3, 4096), (2, 8193), (3, 32003), (2, 129280), (1, 248320), (2, 131071)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tau", [1.0, 0.7])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_token_logprobs(cuda, rows, vocab, dtype, tau):
    from b2g import autograd as ag

    logits, target = _rows(rows, vocab, dtype, vocab + rows)
    if rows > 2:
        target[1] = -100
    live = target != -100
    x64 = logits.double().requires_grad_(True)
    want = ref.logprobs(x64, target, tau)
    for out in (torch.float32, torch.float64):
        x = logits.to(cuda).requires_grad_(True)
        logp = ag.token_logprobs(x, target.to(cuda), temperature=tau, dtype=out)
        assert logp.dtype == out
        off = (logp.detach().cpu().double() - want.detach()).abs()
        assert bool((off <= _logp_tol(want.detach(), vocab, out)).all()), float(off.max())
        assert bool((logp.detach().cpu()[~live] == 0).all())
        g = torch.randn(rows, generator=torch.Generator().manual_seed(3), dtype=torch.float64).to(out)
        (grad,) = torch.autograd.grad(logp, x, g.to(cuda))
        assert grad.dtype == dtype
        _check_cotangent(grad, logits, target, g.double(), g.double().abs() * 2.0 ** -22, tau, dtype, live)


def _policy_case(n, logp, seed):
    g = torch.Generator().manual_seed(seed)
    old = (logp + torch.randn(n, generator=g) * 0.3).float()
    return old, (logp + torch.randn(n, generator=g) * 0.3).float(), torch.randn(n, generator=g), torch.rand(n, generator=g) + 0.25


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", SHAPES + [(64, 257)])
@pytest.mark.parametrize("mode", ["all", "bare", "in place"])
def test_policy_loss(cuda, rows, vocab, dtype, mode):
    from b2g import ops

    tau = 1.0 if mode == "bare" else 0.8
    logits, target = _rows(rows, vocab, dtype, 7 * vocab + rows)
    if rows > 2:
        target[rows // 2] = -100
    live = target != -100
    logp = ref.logprobs(logits.double(), target, tau)
    old, rf, adv, w = _policy_case(rows, logp, vocab)
    if rows > 4:
        w[0] = 0.0
    kw = {} if mode == "bare" else dict(old_logp=old, ref_logp=rf, weight=w, clip_low=0.2, clip_high=0.28, kl_coef=0.1)
    on = {k: v.to(cuda) if torch.is_tensor(v) else v for k, v in kw.items()}
    x = logits.to(cuda)
    keep = x.clone()
    loss, lp, kl, grad = ops.policy_loss(x, target.to(cuda), adv.to(cuda), temperature=tau, out=x if mode == "in place" else None, **on)
    if mode == "in place":
        assert grad is x
    else:
        assert torch.equal(x, keep)
    if mode == "bare":
        want, want_kl, slope = ref.policy(logp, adv, live=live)
        takes = live
    else:
        want, want_kl, slope = ref.policy(logp, adv, old, rf, w, 0.2, 0.28, 0.1, live)
        takes = live & (w != 0)
    tol = _logp_tol(logp, vocab, torch.float64)
    ratio = torch.exp(logp - old.double()) if mode != "bare" else torch.ones_like(logp)
    d = (rf.double() - logp).abs() if mode != "bare" else torch.zeros_like(logp)
    weight = w.double() if mode != "bare" else torch.ones_like(logp)
    # first order in the log-probability's error, and the settings' rounding to 32 bits
    near = (ratio * adv.double()).abs() + 0.1 * torch.exp(d)
    loss_tol = weight * near * (tol + 2.0 ** -23) + want.abs() * 2.0 ** -22
    assert bool(((loss.cpu().double() - want).abs() <= loss_tol)[takes].all())
    assert bool(((lp.cpu().double() - logp).abs() <= _logp_tol(logp, vocab))[takes].all())
    kl_tol = torch.expm1(d).abs() * tol + tol * tol + want_kl.abs() * 2.0 ** -23 + 1e-15
    assert bool(((kl.cpu().double() - want_kl).abs() <= kl_tol)[takes].all())
    for t in (loss, lp, kl):
        assert bool((t.cpu()[~takes] == 0).all())
    _check_cotangent(grad, logits, target, slope, loss_tol + slope.abs() * 2.0 ** -22, tau, dtype, takes)


def test_clipping_on_both_sides_and_at_the_border(cuda):
    """One row per side of each border, far enough off that no rounding decides; the clipped ones have no gradient."""
    from b2g import ops

    logits, target = _rows(8, 64, torch.float32, 1)
    logp = ref.logprobs(logits.double(), target)
    ratio = torch.tensor([1.3, 1.3, 0.7, 0.7, 1.1, 0.9, 1.19, 0.81], dtype=torch.float64)
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0, 2.0, -2.0, 0.0, 0.0])
    old = (logp - torch.log(ratio)).float()
    loss, _, _, grad = ops.policy_loss(logits.to(cuda), target.to(cuda), adv.to(cuda), old_logp=old.to(cuda))
    want, _, slope = ref.policy(logp, adv, old)
    torch.testing.assert_close(loss.cpu().double(), want, rtol=1e-5, atol=0)
    zero = [0, 3, 6, 7]
    assert bool((grad[zero] == 0).all()) and bool((grad[[1, 2, 4, 5]] != 0).any(1).all())
    assert bool((slope[zero] == 0).all())
    # the first step on fresh data: old is the present log-probability, the ratio 1, nothing is clipped even with empty borders
    _, lp, _, _ = ops.policy_loss(logits.to(cuda), target.to(cuda), adv.to(cuda))
    a = ops.policy_loss(logits.to(cuda), target.to(cuda), adv.to(cuda), clip_low=0.0, clip_high=0.0)
    b = ops.policy_loss(logits.to(cuda), target.to(cuda), adv.to(cuda))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pitch,first", [(1000, 0), (1003, 0), (1024, 8), (1011, 5)])
def test_strides_and_alignments(cuda, dtype, pitch, first):
    """Rows that start anywhere, read and written in place and into buffers of another alignment; nothing beside them is touched."""
    from b2g import ops

    logits, target = _rows(9, 997, dtype, pitch)
    adv = torch.randn(9, generator=torch.Generator().manual_seed(2)).to(cuda)
    t = target.to(cuda)
    logp = ref.logprobs(logits.double(), target)

    def right(loss, lp, grad):
        assert bool(((lp.cpu().double() - logp).abs() <= _logp_tol(logp, 997)).all()) and torch.equal(loss, -adv)
        _check_cotangent(grad, logits, target, -adv.cpu().double(), adv.cpu().double().abs() * 2.0 ** -22, 1.0, dtype, target != -100)

    big = torch.full((9, pitch + first), 7.0, dtype=dtype, device=cuda)
    view = big[:, first:first + 997]
    view.copy_(logits)
    loss, lp, _, grad = ops.policy_loss(view, t, adv)
    right(loss, lp, grad)
    for shift in (0, 1, 3):
        other = torch.full((9, 1100), 7.0, dtype=dtype, device=cuda)
        ops.policy_loss(view, t, adv, out=other[:, shift:shift + 997])
        assert torch.equal(other[:, shift:shift + 997], grad)
        assert bool((other[:, :shift] == 7).all()) and bool((other[:, shift + 997:] == 7).all())
    lp2, stats = ops.token_logprobs(view, t)
    assert torch.equal(lp2, lp)
    back = ops.token_logprobs_bwd(-adv, view, t, stats)
    right(-adv, lp, back)
    keep = view.clone()
    ops.policy_loss(view, t, adv, out=view)
    assert torch.equal(view, grad)
    assert bool((big[:, :first] == 7).all()) and bool((big[:, first + 997:] == 7).all())
    view.copy_(keep)
    ops.token_logprobs_bwd(-adv, view, t, stats, out=view)
    assert torch.equal(view, back) and bool((big[:, :first] == 7).all()) and bool((big[:, first + 997:] == 7).all())


@pytest.mark.parametrize("dtype,vocab", [(torch.bfloat16, 1_000_003), (torch.float32, 500_001)])
def test_vocabulary_beyond_a_clusters_memory(cuda, dtype, vocab):
    from b2g import ops

    logits, target = _rows(2, vocab, dtype, 5)
    target[1] = -100
    logp = ref.logprobs(logits.double(), target)
    adv = torch.tensor([0.5, 1.0])
    x = logits.to(cuda)
    loss, lp, _, grad = ops.policy_loss(x, target.to(cuda), adv.to(cuda))
    assert abs(float(lp[0]) - float(logp[0])) <= float(_logp_tol(logp, vocab)[0]) and float(lp[1]) == 0.0
    _check_cotangent(grad, logits, target, -adv.double(), adv.double() * 2.0 ** -22, 1.0, dtype, target != -100)
    lp2, stats = ops.token_logprobs(x, target.to(cuda))
    assert torch.equal(lp2, lp)
    back = ops.token_logprobs_bwd(-adv.to(cuda), x, target.to(cuda), stats)
    _check_cotangent(back, logits, target, -adv.double(), adv.double() * 2.0 ** -22, 1.0, dtype, target != -100)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_vocabulary_and_rows_that_take_no_part(cuda, dtype):
    from b2g import ops

    logits, target = _rows(8, 3001, dtype, 11)
    low = torch.finfo(dtype).min
    rest = torch.ones(8, 3001, dtype=torch.bool)
    rest[torch.arange(8), target] = False
    logits[0][rest[0] & (torch.arange(3001) > 5)] = float("-inf")      # a handful of tokens allowed
    logits[1][rest[1]] = float("-inf")                                 # the target alone: logp 0, no gradient
    logits[2][rest[2] & (torch.arange(3001) % 2 == 0)] = low
    logits[3] = low                                                    # masked throughout by the lowest value: uniform
    logits[4] = float("nan")
    logits[5] = float("inf")
    target[4] = -100
    weight = torch.ones(8)
    weight[5] = 0.0
    takes = (target != -100) & (weight != 0)
    clean = torch.where(takes[:, None], logits, torch.zeros_like(logits))
    logp = ref.logprobs(clean.double(), target)
    adv = torch.linspace(-1, 1, 8) + 0.05
    nan = torch.full((8,), float("nan"))
    old = torch.where(takes, logp, nan.double()).float()
    a = torch.where(takes, adv, nan)
    loss, lp, kl, grad = ops.policy_loss(logits.to(cuda), target.to(cuda), a.to(cuda), old_logp=old.to(cuda), ref_logp=old.to(cuda),
                                         weight=weight.to(cuda), kl_coef=0.5)
    for t in (loss, lp, kl, grad):
        assert bool(torch.isfinite(t).all()) and bool((t[[4, 5]] == 0).all())
    off = (lp.cpu().double() - logp).abs()[takes]
    assert bool((off <= _logp_tol(logp, 3001)[takes]).all())
    assert float(lp[1]) == 0.0 and bool((grad[1] == 0).all())
    assert abs(float(lp[3]) + math.log(3001)) < 1e-5
    uniform = grad[3].cpu().double()
    coef = float(adv[3].abs())
    off = torch.ones(3001, dtype=torch.bool)
    off[target[3]] = False
    torch.testing.assert_close(uniform[off].abs(), torch.full((3000,), coef / 3001, dtype=torch.float64), rtol=2 * ref.HALF[dtype] + 1e-4, atol=0)
    # the log-probabilities' own gradient on the same rows
    logp2, stats = ops.token_logprobs(logits.to(cuda), target.to(cuda))
    g = torch.where(takes, adv, torch.zeros(8)).to(cuda)
    back = ops.token_logprobs_bwd(g, logits.to(cuda), target.to(cuda), stats)
    assert bool(torch.isfinite(back).all()) and bool((back[[4, 5]] == 0).all()) and bool((back[1] == 0).all())
    # a live row that holds NaN, or nothing at all, says so
    bad = torch.full((2, 40), float("-inf"), dtype=dtype, device=cuda)
    bad[1] = float("nan")
    t = torch.tensor([3, 4], device=cuda)
    assert bool(torch.isnan(ops.token_logprobs(bad, t)[0]).all())
    assert bool(torch.isnan(ops.policy_loss(bad, t, torch.ones(2, device=cuda))[0]).all())


def test_targets_outside_the_vocabulary_are_reported_and_ignored(cuda):
    from b2g import _lib, ops

    logits, target = _rows(5, 100, torch.bfloat16, 13)
    target[1], target[3] = 100, -7
    ones = torch.ones(5, device=cuda)
    for call in (lambda: ops.token_logprobs(logits.to(cuda), target.to(cuda))[0],
                 lambda: ops.policy_loss(logits.to(cuda), target.to(cuda), ones)[0],
                 lambda: ops.policy_loss(logits.to(cuda), target.to(cuda), ones)[3]):
        ops.check_status()
        out = call()
        assert bool((out[[1, 3]] == 0).all()) and bool((out[[0, 2, 4]] != 0).any())
        with pytest.raises(_lib.B2GError, match="902"):
            ops.check_status()
    stats = ops.token_logprobs(logits.to(cuda), target.to(cuda))[1]
    with pytest.raises(_lib.B2GError, match="902"):
        ops.check_status()
    assert bool((ops.token_logprobs_bwd(ones, logits.to(cuda), target.to(cuda), stats)[[1, 3]] == 0).all())
    # another ignore index, and one inside the vocabulary
    a = ops.token_logprobs(logits.to(cuda), target.clamp(0, 99).to(cuda), ignore_index=int(target[0]))[0]
    assert float(a[0]) == 0.0
    ops.check_status()


def test_offsets_beyond_32_bits(cuda):
    """More than 2^31 logits: the last rows must be the ones that were asked for."""
    from b2g import ops

    rows, vocab = 8700, 248320
    assert rows * vocab > 1 << 31
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=cuda)
    tail, target_tail = _rows(3, vocab, torch.bfloat16, 17)
    x[-3:] = tail.to(cuda)
    target = torch.full((rows,), -100, device=cuda)
    target[-3:] = target_tail.to(cuda)
    target[0] = 5
    adv = torch.ones(rows, device=cuda)
    logp, stats = ops.token_logprobs(x, target)
    want = ref.logprobs(tail.double(), target_tail)
    assert bool(((logp[-3:].cpu().double() - want).abs() <= _logp_tol(want, vocab)).all())
    assert abs(float(logp[0]) + math.log(vocab)) < 1e-5
    small = ops.policy_loss(tail.to(cuda), target_tail.to(cuda), adv[:3])
    loss, lp, _, grad = ops.policy_loss(x, target, adv, out=x)
    assert torch.equal(grad[-3:], small[3]) and torch.equal(lp[-3:], small[1])
    assert bool((grad[1:-3:997] == 0).all())


def test_gradient_against_differences(cuda):
    """Central differences of the kernel's own loss in fp32: h = 2^-6, truncation h^2/6 times third derivatives of at most 8 |A|
    (ratio, KL term and softmax together), rounding 2^-21 / h."""
    from b2g import ops

    logits, target = _rows(6, 12, torch.float32, 19, 1.0)
    logp = ref.logprobs(logits.double(), target)
    old, rf, adv, w = _policy_case(6, logp, 23)
    old = (logp + torch.linspace(-0.1, 0.1, 6)).float()                # inside the borders throughout
    args = [t.to(cuda) for t in (target, adv)]
    kw = dict(old_logp=old.to(cuda), ref_logp=rf.to(cuda), weight=w.to(cuda), kl_coef=0.3, clip_low=0.5, clip_high=0.5)
    x = logits.to(cuda)
    grad = ops.policy_loss(x, *args, **kw)[3]
    h = 2.0 ** -6
    for col in range(12):
        step = torch.zeros_like(x)
        step[:, col] = h
        diff = (ops.policy_loss(x + step, *args, **kw)[0].double() - ops.policy_loss(x - step, *args, **kw)[0].double()) / (2 * h)
        bound = (h * h / 6 * 8 + 2.0 ** -21 / h) * (1.0 + adv.abs().double() + 0.3) * w.double()
        assert bool(((diff - grad[:, col].double()).abs().cpu() <= bound).all()), col


# ---- preference loss -------------------------------------------------------------------------------
def _pairs(lengths, seed, lead=0, tail=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    ends = torch.tensor([0] + list(lengths)).cumsum(0) + lead
    n = int(ends[-1]) + tail
    logp = -torch.rand(n, generator=g, dtype=torch.float64).to(dtype) * 6
    rf = (logp.double() + 0.2 * torch.randn(n, generator=g, dtype=torch.float64)).float()
    target = torch.where(torch.rand(n, generator=g) < 0.2, -100, 1)
    return logp, rf, target, ends


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("kind,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.2), ("squared", 0.0)])
@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("lengths", [[1, 1], [0, 3], [0, 0], [5, 257, 1030, 2], [3, 0, 70, 1, 9, 0, 4, 300], [40000, 39999]])
def test_preference_loss(cuda, lengths, average, kind, smoothing, dtype):
    from b2g import autograd as ag

    logp, rf, target, ends = _pairs(lengths, sum(lengths), lead=3, tail=5, dtype=dtype)
    masked = rf.clone()
    masked[target == -100] = float("nan")                              # what stands in ignored places is not looked at
    for with_ref, with_target in ((True, True), (False, False)):
        x64 = logp.double().clone().requires_grad_(True)
        r, t = (rf if with_ref else None), (target if with_target else None)
        want = ref.preference(x64, ends, r, 0.1, smoothing, kind, average, t)
        x = logp.to(cuda)
        if with_target:
            x[(target == -100).to(cuda)] = float("nan")
        x.requires_grad_(True)
        got = ag.preference_loss(x, ends.to(cuda), ref_logp=masked.to(cuda) if with_ref else None, beta=0.1, label_smoothing=smoothing,
                                 loss_type=kind, average=average, target=t.to(cuda) if with_target else None)
        total = float((logp.double().abs().sum() + (rf.double().abs().sum() if with_ref else 0)))
        for a, b in zip(got, want):                                    # sums in 64 bits; beta is rounded to 32
            slope = 0.1 if kind == "sigmoid" else 1.0 + 2 * float(want[0].detach().abs().max().sqrt()) if len(want[0]) else 1.0
            torch.testing.assert_close(a.detach().cpu().double(), b.detach(), rtol=2.0 ** -22, atol=2.0 ** -24 * 40 * slope + total * 1e-14 * slope)
        g = torch.randn(len(lengths) // 2, generator=torch.Generator().manual_seed(1))
        (grad,) = torch.autograd.grad(got[0], x, g.to(cuda))
        (want_grad,) = torch.autograd.grad(want[0], x64, g.double())
        want_grad = torch.zeros_like(logp.double()) if want_grad is None else want_grad
        assert grad.dtype == dtype
        scale = float(g.abs().max()) * (0.1 if kind == "sigmoid" else 10 + 2 * float(want[0].detach().abs().max().sqrt()))
        torch.testing.assert_close(grad.cpu().double(), want_grad, rtol=2.0 ** -21, atol=2.0 ** -22 * scale)
        counted = torch.zeros(len(logp), dtype=torch.bool)
        counted[int(ends[0]):int(ends[-1])] = True
        if with_target:
            counted &= target != -100
        assert bool((grad.cpu()[~counted] == 0).all())


def test_preference_types_of_the_reference(cuda):
    """The reference's log-probabilities in either type: the same numbers give the same result, whatever they are held in."""
    from b2g import ops

    logp, rf, target, ends = _pairs([300, 5, 0, 77], 41)
    on = dict(target=target.to(cuda), average=True)
    for a in (logp, logp.double()):
        got = [ops.preference_loss(a.to(cuda), ends.to(cuda), ref_logp=b.to(cuda), **on) for b in (rf, rf.double())]
        assert all(torch.equal(x, y) for x, y in zip(*got))
    with pytest.raises(TypeError, match="ref_logp"):
        ops.preference_loss(logp.to(cuda), ends.to(cuda), ref_logp=rf.bfloat16().to(cuda))


def test_preference_gradient_against_differences(cuda):
    from b2g import autograd as ag

    logp, rf, target, ends = _pairs([4, 3, 2, 5], 3, dtype=torch.float64)
    x = logp.to(cuda).requires_grad_(True)
    on = dict(ref_logp=rf.to(cuda), target=target.to(cuda))
    for kind in ("sigmoid", "squared"):
        loss, _, _ = ag.preference_loss(x, ends.to(cuda), beta=0.5, loss_type=kind, **on)
        (grad,) = torch.autograd.grad(loss.sum(), x)
        h = 2.0 ** -5
        for i in range(len(logp)):
            step = torch.zeros_like(x)
            step[i] = h
            with torch.no_grad():
                up, down = (ag.preference_loss(x + s, ends.to(cuda), beta=0.5, loss_type=kind, **on)[0].double().sum() for s in (step, -step))
            # third derivative of the sigmoid loss below beta^3 / 8; the square has none; losses are fp32
            assert abs(float((up - down) / (2 * h) - grad[i])) <= h * h / 6 / 8 + 2.0 ** -23 * float(loss.detach().abs().sum() + 1) / h


def test_pairs_of_nothing_and_bad_offsets(cuda):
    from b2g import _lib, autograd as ag, ops

    empty = torch.zeros(0, device=cuda, requires_grad=True)
    loss, chosen, rejected = ag.preference_loss(empty, torch.zeros(3, dtype=torch.int64, device=cuda))
    assert abs(float(loss) - math.log(2)) < 1e-6 and float(chosen) == float(rejected) == 0.0
    assert torch.autograd.grad(loss.sum(), empty)[0].shape == (0,)
    x = torch.ones(6, device=cuda, requires_grad=True)
    loss, _, _ = ag.preference_loss(x, torch.zeros(1, dtype=torch.int64, device=cuda))
    assert loss.shape == (0,) and bool((torch.autograd.grad(loss.sum(), x)[0] == 0).all())
    for bad in ([0, 4, 2], [0, 3, 99], [-5, 2, 4], [7, 8, 9]):
        ops.check_status()
        out = ops.preference_loss(x.detach(), torch.tensor(bad, device=cuda))
        back = ops.preference_loss_bwd(torch.ones(1, device=cuda), out[3], torch.tensor(bad, device=cuda), 6)
        assert bool(torch.isfinite(out[0]).all()) and bool(torch.isfinite(back).all())
        with pytest.raises(_lib.B2GError, match="905"):
            ops.check_status()


def test_streams_and_captured_graph(cuda):
    from b2g import ops

    logits, target = _rows(40, 5003, torch.bfloat16, 29)
    x, t = logits.to(cuda), target.to(cuda)
    adv = torch.randn(40, device=cuda)
    ends = torch.tensor([0, 9, 20, 31, 40], device=cuda)

    def step():
        logp, stats = ops.token_logprobs(x, t, dtype=torch.float64)
        loss, chosen, rejected, coef = ops.preference_loss(logp, ends)
        g = ops.preference_loss_bwd(torch.ones(2, device=cuda), coef, ends, 40, dtype=torch.float64)
        return (logp, stats, loss, chosen, rejected, g, ops.token_logprobs_bwd(g, x, t, stats)) + ops.policy_loss(x, t, adv, old_logp=logp.float())

    want = step()
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for s in (first, second):                                          # two at once
        with torch.cuda.stream(s):
            outs.append(step())
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    other, _ = _rows(40, 5003, torch.bfloat16, 31)
    x.copy_(other)
    adv.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_refusals(cuda):
    from b2g import ops

    x, t, a = torch.zeros(4, 16, device=cuda), torch.zeros(4, dtype=torch.int64, device=cuda), torch.zeros(4, device=cuda)
    with pytest.raises(TypeError, match="bf16 or fp32"):
        ops.policy_loss(x.half(), t, a)
    with pytest.raises(RuntimeError, match="stride"):
        ops.token_logprobs(torch.zeros(16, 4, device=cuda).t(), t)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.policy_loss(x[:1].expand(4, 16), t, a)
    with pytest.raises(TypeError, match="target"):
        ops.policy_loss(x, t.int(), a)
    with pytest.raises(ValueError, match="advantage"):
        ops.policy_loss(x, t, a[:3])
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.policy_loss(x, t, torch.zeros(8, device=cuda)[::2])
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.policy_loss(x, t, a.cpu())
    for kw, what in ((dict(temperature=0.0), "temperature"), (dict(temperature=float("inf")), "temperature"), (dict(clip_low=1.5), "clip_low"),
                     (dict(clip_high=-0.1), "clip_high"), (dict(kl_coef=0.1), "ref_logp"), (dict(kl_coef=-1.0, ref_logp=a), "kl_coef"),
                     (dict(out=x.bfloat16()), "out must match"), (dict(out=torch.zeros(4, 15, device=cuda)), "out must match")):
        with pytest.raises(ValueError, match=what):
            ops.policy_loss(x, t, a, **kw)
    buf = torch.zeros(100, device=cuda)
    with pytest.raises(ValueError, match="overlaps"):
        ops.policy_loss(buf[:64].view(4, 16), t, a, out=buf[8:72].view(4, 16))
    with pytest.raises(TypeError, match="fp32 or fp64"):
        ops.token_logprobs(x, t, dtype=torch.bfloat16)
    ends = torch.tensor([0, 2, 4], device=cuda)
    for kw, what in ((dict(beta=0.0), "beta"), (dict(label_smoothing=0.5), "label_smoothing"), (dict(loss_type="hinge"), "loss_type"),
                     (dict(loss_type="squared", label_smoothing=0.1), "label_smoothing")):
        with pytest.raises(ValueError, match=what):
            ops.preference_loss(a, ends, **kw)
    with pytest.raises(ValueError, match="offsets"):
        ops.preference_loss(a, ends[:2])
    with pytest.raises(TypeError, match="fp32 or fp64"):
        ops.preference_loss(a.bfloat16(), ends)
    tau = C.c_float(1.0)
    from b2g import _lib
    assert _lib.load().b2g_token_logprobs(None, 16, 0, None, None, 0, None, 4, 16, tau, -100, None, None) == -1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [3000, 20001, 130003])
def test_maxima_that_no_sample_sees(cuda, dtype, vocab):
    """One logit far above everything else, at a column of its own in every row: sums taken against too low a reference must
    overflow unnoticed or be made again.  Among the rows are a NaN, a +inf, a row of -inf but for the target, one masked
    throughout by the type's lowest value, and ignored ones between them."""
    from b2g import ops

    logits, target = _rows(24, vocab, dtype, vocab)
    for r in range(24):
        logits[r, (r * 7919 + 5) % vocab] = 20.0 + 12.0 * r                # 20 ... 296
    logits[3] = torch.finfo(dtype).min
    logits[7] = float("-inf")
    logits[7, target[7]] = 1.5
    logits[11, 17] = float("nan")
    logits[13, 19] = float("inf")
    target[[5, 12, 20]] = -100
    takes = target != -100
    whole = takes.clone()
    whole[[11, 13]] = False
    clean = torch.where(whole[:, None], logits, torch.zeros_like(logits))
    logp = ref.logprobs(clean.double(), target)
    adv = torch.linspace(-1, 1, 24) + 0.01
    x, t = logits.to(cuda), target.to(cuda)
    for tau in (1.0, 3.0):
        logp = ref.logprobs(clean.double(), target, tau)
        got, stats = ops.token_logprobs(x, t, tau, dtype=torch.float64)
        assert bool(torch.isnan(got[[11, 13]]).all()) and bool((got[[5, 12, 20]] == 0).all())
        off = (got.cpu() - logp).abs()[whole]
        assert bool((off <= ref.lse_error(vocab) + logp.abs()[whole] * 2.0 ** -50).all()), float(off.max())
        loss, lp, _, grad = ops.policy_loss(x, t, adv.to(cuda), temperature=tau)
        assert bool(torch.isnan(loss[[11, 13]]).all())
        assert bool(((lp.cpu().double() - logp).abs() <= _logp_tol(logp, vocab))[whole].all())
        back = ops.token_logprobs_bwd(-adv.to(cuda), x, t, stats, tau)
        for g in (grad, back):
            g = g.clone()
            g[[11, 13]] = 0
            _check_cotangent(g[whole.to(cuda)], clean[whole], target[whole], -adv.double()[whole], adv.double().abs()[whole] * 2.0 ** -22, tau, dtype,
                             target[whole] != -100)


def test_many_rows_of_every_path_repeat_bit_for_bit(cuda):
    """More rows than clusters, ignored ones among them, several times over: the pipeline's order does not show."""
    from b2g import ops

    for vocab, rows in ((1001, 900), (9000, 700), (40003, 400), (129280, 200)):
        g = torch.Generator(device=cuda).manual_seed(vocab)
        x = (torch.randn(rows, vocab, generator=g, device=cuda) * 2).bfloat16()
        t = torch.randint(0, vocab, (rows,), generator=g, device=cuda)
        t[torch.rand(rows, generator=g, device=cuda) < 0.3] = -100
        t[rows // 2:rows // 2 + 40] = -100
        adv = torch.randn(rows, generator=g, device=cuda)
        want = ops.policy_loss(x, t, adv)
        logp = ops.token_logprobs(x, t)[0]
        # wide rows have a kernel of their own for either: twice the error of a log-sum-exp, and half a step on both sides
        assert bool(((logp - want[1]).abs().double() <= 2 * ref.lse_error(vocab) + 2.0 ** -23 * logp.abs().double()).all())
        for _ in range(3):
            got = ops.policy_loss(x, t, adv)
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(ops.token_logprobs(x, t)[0], logp)
        some = torch.randint(0, rows, (12,)).tolist()
        for r in some:                                                   # a row's result does not depend on its neighbours
            one = ops.policy_loss(x[r:r + 1], t[r:r + 1], adv[r:r + 1])
            assert torch.equal(one[1], want[1][r:r + 1]) or abs(float(one[1] - want[1][r])) <= 2 * ref.lse_error(vocab)
            torch.testing.assert_close(one[3].float(), want[3][r:r + 1].float(), rtol=2.0 ** -7, atol=1e-6)


def test_results_are_changed_in_place_like_any_tensor(cuda):
    from b2g import autograd as ag

    logp, _, target, ends = _pairs([4, 3, 2, 5], 5, dtype=torch.float32)
    x = logp.to(cuda).requires_grad_(True)
    plain, _, _ = ag.preference_loss(x, ends.to(cuda), target=target.to(cuda))
    (want,) = torch.autograd.grad((plain * 3.0 * plain.detach() * 3.0).sum(), x)
    loss, chosen, rejected = ag.preference_loss(x, ends.to(cuda), target=target.to(cuda))
    loss.mul_(3.0)
    y = (loss * loss.detach().clone()).sum()
    chosen.neg_()
    rejected.zero_()
    (got,) = torch.autograd.grad(y, x)
    # the same products in another order: four roundings of fp32 on either side
    assert bool(((got - want).abs() <= 8 * 2.0 ** -24 * want.abs()).all())


def test_tokens_that_cannot_occur(cuda):
    """A sequence with a token of probability 0: the loss is 0 where it is the rejected one, infinite where it is the chosen one."""
    from b2g import ops

    logp = torch.tensor([-1.0, -2.0, -math.inf, -3.0, -0.5, -math.inf, -2.0, -1.0], device=cuda)
    ends = torch.tensor([0, 2, 4, 6, 8], device=cuda)       # chosen: finite, impossible; rejected: impossible, finite
    loss, chosen, rejected, coef = ops.preference_loss(logp, ends)
    assert loss.tolist() == [0.0, math.inf] and rejected[0] == -math.inf and chosen[1] == -math.inf
    grad = ops.preference_loss_bwd(torch.ones(2, device=cuda), coef, ends, 8)
    beta = float(torch.tensor(0.1))
    assert grad.tolist() == [0.0, 0.0, -beta, -beta, 0.0, 0.0, beta, beta]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(900, 700), (700, 9001), (450, 50001), (90, 260003), (3, 130003)])
def test_rows_that_take_no_part_change_no_other(cuda, dtype, rows, vocab):
    """Ignored rows before, behind, between and instead of all others: the rest is the same bit for bit, the ignored ones are 0."""
    from b2g import ops

    g = torch.Generator(device=cuda).manual_seed(vocab)
    x = torch.randn(rows, vocab, device=cuda, generator=g).to(dtype)
    target = torch.randint(0, vocab, (rows,), device=cuda, generator=g)
    adv = torch.randn(rows, device=cuda, generator=g)
    every = ops.token_logprobs(x, target, dtype=torch.float64)[0]
    loss, logp, _, grad = ops.policy_loss(x, target, adv)
    at = torch.arange(rows, device=cuda)
    for dead in (at < rows // 2, at >= rows // 3, at % 3 != 1, at % 7 == 0, at >= 0):
        t = torch.where(dead, -100, target)
        got = ops.token_logprobs(x, t, dtype=torch.float64)[0]
        assert torch.equal(got, torch.where(dead, 0.0, every))
        l, lp, _, gr = ops.policy_loss(x, t, adv)
        assert torch.equal(l, torch.where(dead, 0.0, loss)) and torch.equal(lp, torch.where(dead, 0.0, logp))
        assert torch.equal(gr, torch.where(dead[:, None], torch.zeros((), dtype=dtype, device=cuda), grad))
    ops.check_status()
