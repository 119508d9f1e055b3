"""GPU: the post-training losses on a packed LM head, and one whole step through router, experts, head and policy loss.

The oracle multiplies the dequantised head in fp32 and rounds the logits to bf16 as the packed product does.  Two products that
round to bf16 in another order differ by a step of 2^-7 in few logits; relative L2 <= 1e-2 on gradients and 2e-2 absolute on a
log-probability are the bars of the supervised packed loss (test_lm_head_loss_gpu.py)."""
import numpy as np
import pytest
import torch

from oracle import dense_ref, gguf_oracle as go, posttrain_ref as ref

pytestmark = pytest.mark.gpu


def _head(cuda, vocab, hidden, qtype, seed):
    from b2g.gguf_types import GGUFLinear, GGUFQuantizedTensor

    payload = go.quantize((np.random.default_rng(seed).standard_normal((vocab, hidden)) * 0.08).astype(np.float32), qtype)
    head = GGUFLinear(hidden, vocab)
    head.weight = GGUFQuantizedTensor(torch.from_numpy(payload).to(cuda), quant_type=qtype, logical_shape=(vocab, hidden))
    return head, dense_ref.dequant_bf16(payload, qtype)


def _case(vocab, hidden, rows, seed):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(rows, hidden, generator=g).bfloat16()
    target = torch.randint(0, vocab, (rows,), generator=g)
    target[::7] = -100
    return g, h, target


def _logits(h, w):
    return (h.float() @ w.float().t()).bfloat16().double()


@pytest.mark.parametrize("qtype,vocab,hidden,rows,chunk", [(go.Q8_0, 37, 256, 34, 2048), (go.Q6_K, 1032, 2048, 300, 128), (go.Q4_K, 4096, 512, 130, 64)])
def test_log_probabilities_and_policy_loss(cuda, qtype, vocab, hidden, rows, chunk):
    import gguf_policy_loss as gp

    head, w = _head(cuda, vocab, hidden, qtype, vocab)
    g, h, target = _case(vocab, hidden, rows, vocab)
    live = target != -100
    x64 = _logits(h, w)
    want = ref.logprobs(x64, target, 0.9)
    cot = torch.randn(rows, generator=g)
    hc = h.to(cuda).requires_grad_(True)
    logp = gp.packed_token_logprobs(hc, head, target.to(cuda), temperature=0.9, chunk_size=chunk)
    assert float((logp.detach().cpu().double() - want).abs().max()) < 2e-2
    logp.backward(cot.to(cuda))
    p = torch.softmax(x64 / 0.9, 1)
    hot = torch.zeros_like(p)
    hot[torch.arange(rows), target.clamp(min=0)] = 1.0
    onehot_minus_p = torch.where(live[:, None], hot - p, torch.zeros_like(p))
    assert dense_ref.rel_l2(hc.grad, (cot.double()[:, None] * onehot_minus_p / 0.9) @ w.double()) < 1e-2
    with torch.no_grad():
        assert torch.equal(gp.packed_token_logprobs(hc, head, target.to(cuda), temperature=0.9, chunk_size=chunk), logp)
        assert gp.packed_token_logprobs(hc.reshape(1, rows, hidden), head, target.to(cuda)[None]).shape == (1, rows)

    # far from the clipping borders on either side, so that a logit's rounding decides nothing
    ratio = torch.tensor([1.05, 1.6, 0.6, 0.95])[torch.arange(rows) % 4]
    old = (want - torch.log(ratio.double())).float()
    rf = (want + 0.1 * torch.randn(rows, generator=g, dtype=torch.float64)).float()
    adv, weight = torch.randn(rows, generator=g), torch.full((rows,), 1.0 / rows)
    hc2 = h.to(cuda).requires_grad_(True)
    loss, lp, kl = gp.packed_policy_loss(hc2, head, target.to(cuda), adv.to(cuda), old_logp=old.to(cuda), ref_logp=rf.to(cuda), weight=weight.to(cuda),
                                         kl_coef=0.1, temperature=0.9, chunk_size=chunk)
    (loss * 3.0).backward()
    want_loss, _, slope = ref.policy(want, adv, old, rf, weight, 0.2, 0.2, 0.1, live)
    assert abs(float(loss) - float(want_loss.sum())) < 2e-2
    assert torch.equal(lp, logp.detach()) and not lp.requires_grad and kl.shape == target.shape
    assert dense_ref.rel_l2(hc2.grad, 3.0 * (slope[:, None] * onehot_minus_p / 0.9) @ w.double()) < 2e-2
    assert head.weight.grad is None
    # without a gradient the input-gradient product is not made
    with torch.no_grad():
        again, _, _ = gp.packed_policy_loss(hc2, head, target.to(cuda), adv.to(cuda), old_logp=old.to(cuda), ref_logp=rf.to(cuda),
                                            weight=weight.to(cuda), kl_coef=0.1, temperature=0.9, chunk_size=chunk)
    assert torch.equal(again, loss.detach())


@pytest.mark.parametrize("kind,average", [("sigmoid", False), ("squared", True)])
def test_preference_loss_on_a_packed_head(cuda, kind, average):
    import gguf_policy_loss as gp

    vocab, hidden, rows = 1032, 2048, 90
    head, w = _head(cuda, vocab, hidden, go.Q6_K, 3)
    g, h, target = _case(vocab, hidden, rows, 4)
    ends = torch.tensor([0, 20, 41, 41, 83])
    hf = h.double().requires_grad_(True)
    x = hf @ w.double().t()
    rf = (ref.logprobs(_logits(h, w), target) + 0.1 * torch.randn(rows, generator=g, dtype=torch.float64)).float()
    want, wc, wr = ref.preference(ref.logprobs(x, target), ends, rf, 0.1, 0.0, kind, average, target)
    want.sum().backward()
    hc = h.to(cuda).requires_grad_(True)
    loss, chosen, rejected = gp.packed_preference_loss(hc, head, target.to(cuda), ends.to(cuda), ref_logp=rf.to(cuda), loss_type=kind, average=average,
                                                       chunk_size=64)
    loss.sum().backward()
    for a, b in ((chosen, wc), (rejected, wr)):
        assert float((a.cpu().double() - b.detach()).abs().max()) < 0.1 * 42 * 2e-2
    assert dense_ref.rel_l2(hc.grad, hf.grad) < 3e-2
    assert bool((hc.grad[83:] == 0).all())


def test_refusals(cuda):
    import gguf_policy_loss as gp

    head, _ = _head(cuda, 64, 256, go.Q8_0, 5)
    h = torch.zeros(3, 256, device=cuda, dtype=torch.bfloat16)
    t, a = torch.zeros(3, dtype=torch.int64, device=cuda), torch.zeros(3, device=cuda)
    with pytest.raises(TypeError, match="BF16 hidden"):
        gp.packed_token_logprobs(h.float(), head, t)
    with pytest.raises(ValueError, match="Targets"):
        gp.packed_token_logprobs(h, head, t[:2])
    with pytest.raises(ValueError, match="Hidden size"):
        gp.packed_token_logprobs(h[:, :128], head, t)
    with pytest.raises(ValueError, match="old_logp"):
        gp.packed_policy_loss(h, head, t, a, old_logp=a[:2])
    with pytest.raises(ValueError, match="chunk_size"):
        gp.packed_token_logprobs(h, head, t, chunk_size=0)
    with pytest.raises(ValueError, match="one behind the other"):
        gp.packed_preference_loss(h[None], head, t[None], torch.tensor([0, 1, 3], device=cuda))
    head.compute_dtype = torch.float16
    with pytest.raises(RuntimeError, match="BF16 compute_dtype"):
        gp.packed_policy_loss(h, head, t, a)


def test_a_post_training_step_through_router_experts_and_head(cuda):
    """Router -> packed experts -> packed head -> policy loss and back: the gradients of router, adapters and hidden states are
    there, finite, and the router's is that of the weights' path (compared with elementary autograd on the same choice)."""
    import gguf_policy_loss as gp
    from b2g import ops
    from b2g.routing import build_plan, combine
    from fast_moe_ranking import route_experts

    tokens, hidden, experts, inter, top_k, vocab = 200, 2048, 16, 256, 4, 1032
    rng = np.random.default_rng(1)
    g = torch.Generator().manual_seed(1)

    def packed(rows, cols):
        return torch.from_numpy(go.quantize((rng.standard_normal((rows, cols)) * 0.03).astype(np.float32), go.Q4_K)).to(cuda)

    up, down = packed(experts * inter, hidden), packed(experts * hidden, inter)
    head, _ = _head(cuda, vocab, hidden, go.Q6_K, 7)
    x = torch.randn(tokens, hidden, generator=g).bfloat16().to(cuda).requires_grad_(True)
    gate = (torch.randn(experts, hidden, generator=g) * 0.03).bfloat16().to(cuda).requires_grad_(True)
    bias = (torch.randn(experts, generator=g) * 0.05).to(cuda)
    target = torch.randint(0, vocab, (tokens,), generator=g).to(cuda)
    target[::9] = -100
    adv = torch.randn(tokens, generator=g).to(cuda)

    def block(route):
        w, idx = route(torch.nn.functional.linear(x, gate))
        plan = build_plan(x, idx, w, experts)
        ids = torch.arange(experts, device=cuda)
        y = torch.ops.b2g.grouped_mmq(plan.selected_hidden_states, up, ids, plan.group_offsets, go.Q4_K, inter)
        z = torch.ops.b2g.grouped_mmq(torch.nn.functional.silu(y), down, ids, plan.group_offsets, go.Q4_K, hidden)
        return x + combine(z, plan), idx

    kw = dict(correction_bias=bias, score_function="sigmoid", num_groups=4, top_groups=2, renormalize=True, scaling_factor=2.5)
    out, idx = block(lambda logits: route_experts(logits, top_k, **kw))
    loss, _, _ = gp.packed_policy_loss(out, head, target, adv, weight=torch.full((tokens,), 1.0 / tokens, device=cuda))
    grads = torch.autograd.grad(loss, (x, gate))
    assert all(bool(torch.isfinite(v).all()) and float(v.float().norm()) > 0 for v in grads)

    def plain(logits):
        s = torch.sigmoid(logits.float()).gather(1, idx)
        return 2.5 * s / s.sum(1, keepdim=True), idx

    out2, _ = block(plain)
    loss2, _, _ = gp.packed_policy_loss(out2, head, target, adv, weight=torch.full((tokens,), 1.0 / tokens, device=cuda))
    want = torch.autograd.grad(loss2, (x, gate))
    assert abs(float(loss) - float(loss2)) < 1e-3
    for a, b in zip(grads, want):
        assert dense_ref.rel_l2(a, b.cpu().double()) < 1e-2
    ops.check_status()


def test_the_gradient_is_scaled_in_32_bits(cuda):
    import gguf_policy_loss as gp

    head, _ = _head(cuda, 1032, 2048, go.Q6_K, 5)
    g, h, target = _case(1032, 2048, 40, 6)
    adv = torch.randn(40, generator=g).to(cuda)

    def grad(scale):
        x = h.to(cuda).requires_grad_(True)
        (gp.packed_policy_loss(x, head, target.to(cuda), adv)[0] * scale).backward()
        return x.grad

    third = torch.tensor(1.0 / 3.0)
    assert torch.equal(grad(float(third)), (grad(1.0).float() * third.to(cuda)).bfloat16())
