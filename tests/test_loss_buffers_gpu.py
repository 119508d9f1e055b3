"""GPU: buffers that the row losses write to: what autograd has saved, and columns beside the logits in one tensor."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _case(cuda, rows=6, vocab=501, dtype=torch.float32):
    g = torch.Generator(device=cuda).manual_seed(rows + vocab)
    logits = torch.randn(rows, vocab, generator=g, device=cuda).to(dtype)
    target = torch.randint(0, vocab, (rows,), generator=g, device=cuda)
    return logits, target, torch.randn(rows, generator=g, device=cuda)


def test_logits_that_a_graph_has_saved(cuda):
    """Overwriting them is an in-place change like any other: the backward pass that needs them says so."""
    from b2g import autograd as ag, ops

    logits, target, adv = _case(cuda)
    x = (logits.clone().requires_grad_(True)) * 1.0
    logp = ag.token_logprobs(x, target)
    ops.policy_loss(x, target, adv, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        logp.sum().backward()
    x = (logits.clone().requires_grad_(True)) * 1.0
    logp = ag.token_logprobs(x, target)
    stats = ops.token_logprobs(x, target)[1]
    ops.token_logprobs_bwd(adv, x, target, stats, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        logp.sum().backward()
    # a buffer of the caller's, saved by somebody else
    buf = torch.ones_like(logits)
    w = torch.ones((), device=cuda, requires_grad=True)
    y = (buf * w).sum()
    ops.policy_loss(logits, target, adv, out=buf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    # without an `out` nothing of the caller's changes
    x = (logits.clone().requires_grad_(True)) * 1.0
    logp = ag.token_logprobs(x, target)
    grad = ops.policy_loss(x, target, adv)[3]
    logp.sum().backward()
    # and logits that nobody has saved take their own gradient back, as the packed head does
    leaf = logits.clone().requires_grad_(True)
    x = leaf * 1.0
    out = ops.policy_loss(x, target, adv, out=x.detach())[3]
    x.backward(out)
    assert torch.equal(leaf.grad, grad)


def test_inference_tensors(cuda):
    from b2g import ops

    with torch.inference_mode():
        logits, target, adv = _case(cuda)
        want = ops.policy_loss(logits, target, adv)[3]
        assert torch.equal(ops.policy_loss(logits, target, adv, out=logits)[3], want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(5, 501), (3, 9001), (3, 40001), (7, 64)])
def test_columns_beside_the_logits(cuda, dtype, rows, vocab):
    """Logits and gradient side by side in one tensor share no element, in either order; one column of overlap is refused."""
    from b2g import ops

    logits, target, adv = _case(cuda, rows, vocab, dtype)
    for first, second in ((0, vocab), (0, vocab + 3), (vocab + 1, 0), (vocab, 0), (2, vocab + 2)):
        both = torch.full((rows, 2 * vocab + 5), 7.0, dtype=dtype, device=cuda)
        x, out = both[:, first:first + vocab], both[:, second:second + vocab]
        x.copy_(logits)
        # of the same rows: which terms share a 16-byte vector, and so the order of the sum, goes by where the logits lie
        want = ops.policy_loss(x, target, adv)[3]
        assert ops.policy_loss(x, target, adv, out=out)[3] is out
        assert torch.equal(out, want) and torch.equal(x, logits)
        kept = torch.ones(2 * vocab + 5, dtype=torch.bool, device=cuda)
        kept[first:first + vocab] = False
        kept[second:second + vocab] = False
        assert bool((both[:, kept] == 7).all())
        stats = ops.token_logprobs(x, target)[1]
        apart = ops.token_logprobs_bwd(adv, x, target, stats)
        assert torch.equal(ops.token_logprobs_bwd(adv, x, target, stats, out=out), apart)
    both = torch.zeros(rows, 2 * vocab, dtype=dtype, device=cuda)
    for first, second in ((0, vocab - 1), (vocab - 1, 0), (0, 1), (1, 0)):
        with pytest.raises(ValueError, match="overlaps"):
            ops.policy_loss(both[:, first:first + vocab], target, adv, out=both[:, second:second + vocab])
    # rows of another pitch, and rows that wrap into the next one's columns
    flat = torch.zeros(rows * (2 * vocab + 1) + vocab, dtype=dtype, device=cuda)
    a = flat.as_strided((rows, vocab), (2 * vocab, 1), 0)
    with pytest.raises(ValueError, match="overlaps"):
        ops.policy_loss(a, target, adv, out=flat.as_strided((rows, vocab), (2 * vocab + 1, 1), vocab))
    with pytest.raises(ValueError, match="overlaps"):
        ops.policy_loss(a, target, adv, out=flat.as_strided((rows, vocab), (2 * vocab, 1), vocab + 1))
