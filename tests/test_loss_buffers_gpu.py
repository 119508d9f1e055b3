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
