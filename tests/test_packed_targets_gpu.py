"""GPU: targets outside the vocabulary on the packed head take no part in any of its losses, and are reported."""
import numpy as np
import pytest
import torch

from oracle import gguf_oracle as go

pytestmark = pytest.mark.gpu


def _head(cuda, vocab, hidden):
    from b2g.gguf_types import GGUFLinear, GGUFQuantizedTensor

    payload = go.quantize((np.random.default_rng(1).standard_normal((vocab, hidden)) * 0.08).astype(np.float32), go.Q8_0)
    head = GGUFLinear(hidden, vocab)
    head.weight = GGUFQuantizedTensor(torch.from_numpy(payload).to(cuda), quant_type=go.Q8_0, logical_shape=(vocab, hidden))
    return head


@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("ignore", [-100, 3])
def test_preference_loss(cuda, average, ignore):
    """The same as with those targets ignored, bit for bit, whatever the reference's log-probabilities hold in their places."""
    import gguf_policy_loss as gp
    from b2g import _lib, ops

    vocab, hidden = 300, 256
    head = _head(cuda, vocab, hidden)
    g = torch.Generator().manual_seed(2)
    h = torch.randn(40, hidden, generator=g).bfloat16().to(cuda)
    target = torch.randint(4, vocab, (40,), generator=g)
    target[[2, 17, 30]] = ignore
    rf = (-torch.rand(40, generator=g) * 6).to(cuda)
    ends = torch.tensor([0, 9, 18, 30, 40], device=cuda)
    bad = target.clone()
    bad[[4, 11, 12, 25, 39]] = torch.tensor([vocab, -7, 1 << 40, vocab + 5, -1])
    clean = torch.where((bad >= 0) & (bad < vocab), bad, ignore)

    def run(t):
        x = h.clone().requires_grad_(True)
        out = gp.packed_preference_loss(x, head, t.to(cuda), ends, ref_logp=rf, average=average, ignore_index=ignore)
        out[0].sum().backward()
        return (*out, x.grad)

    ops.check_status()
    want = run(clean)
    ops.check_status()
    got = run(bad)
    with pytest.raises(_lib.B2GError, match="902"):
        ops.check_status()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_log_probabilities_and_policy_loss(cuda):
    import gguf_policy_loss as gp
    from b2g import _lib, ops

    head = _head(cuda, 300, 256)
    g = torch.Generator().manual_seed(3)
    h = torch.randn(12, 256, generator=g).bfloat16().to(cuda)
    target = torch.randint(0, 300, (12,), generator=g).to(cuda)
    bad = target.clone()
    bad[3], bad[8] = 300, -5
    adv = torch.randn(12, generator=g).to(cuda)
    x = h.clone().requires_grad_(True)
    logp = gp.packed_token_logprobs(x, head, bad)
    (grad,) = torch.autograd.grad(logp.sum(), x)
    assert bool((logp[[3, 8]] == 0).all()) and bool((grad[[3, 8]] == 0).all())
    loss, lp, kl = gp.packed_policy_loss(x, head, bad, adv, ref_logp=torch.zeros(12, device=cuda), kl_coef=0.1)
    (grad,) = torch.autograd.grad(loss, x)
    assert bool((lp[[3, 8]] == 0).all()) and bool((kl[[3, 8]] == 0).all()) and bool((grad[[3, 8]] == 0).all())
    with pytest.raises(_lib.B2GError, match="902"):
        ops.check_status()
