"""CPU: the routing and post-training entry points refuse bad arguments before they touch a device."""
import ctypes as C

import pytest
import torch

f = C.c_float


@pytest.mark.parametrize("args,what", [
    ((None, 513, 1, None, 0, 1, 1, 1, 1, f(1.0), None, None, 4, 513, 8, None), b"513 experts"),
    ((None, 64, 1, None, 0, 1, 1, 1, 1, f(1.0), None, None, 4, 64, 33, None), b"top_k=33"),
    ((None, 64, 1, None, 0, 1, 1, 1, 1, f(1.0), None, None, 4, 64, 0, None), b"top_k=0"),
    ((None, 64, 2, None, 0, 1, 1, 1, 1, f(1.0), None, None, 4, 64, 8, None), b"logits_dtype"),
    ((None, 64, 1, None, 3, 1, 1, 1, 1, f(1.0), None, None, 4, 64, 8, None), b"score_fn"),
    ((None, 64, 1, None, 0, 1, 1, 1, 1, f(0.0), None, None, 4, 64, 8, None), b"scaling"),
    ((None, 64, 1, None, 0, 1, 1, 1, 1, f(float("nan")), None, None, 4, 64, 8, None), b"scaling"),
    ((None, 63, 1, None, 0, 1, 1, 1, 1, f(1.0), None, None, 4, 64, 8, None), b"row pitch"),
    ((None, 64, 1, None, 0, 1, 1, 1, 1, f(1.0), None, None, 4, 64, 8, None), b"null"),
    ((None, 64, 1, None, 0, 7, 1, 1, 1, f(1.0), None, None, 0, 64, 8, None), b"7 groups"),
    ((None, 64, 1, None, 0, 64, 1, 1, 1, f(1.0), None, None, 0, 64, 1, None), b"64 groups"),
    ((None, 64, 1, None, 0, 8, 9, 1, 1, f(1.0), None, None, 0, 64, 8, None), b"top_groups=9"),
    ((None, 64, 1, None, 0, 8, 1, 1, 1, f(1.0), None, None, 0, 64, 9, None), b"kept groups"),
    ((None, 64, 1, None, 0, 8, 2, 3, 1, f(1.0), None, None, 0, 64, 8, None), b"group_experts"),
    ((None, 64, 1, None, 0, 1, 1, 1, 1, f(1.0), None, None, -1, 64, 8, None), b"token count")])
def test_route_experts_entry(lib, args, what):
    assert lib.b2g_route_experts(*args) == -1 and what in lib.b2g_last_error()


def test_no_rows_is_no_work(lib):
    assert lib.b2g_route_experts(None, 64, 1, None, 0, 1, 1, 1, 1, f(1.0), None, None, 0, 64, 8, None) == 0
    assert lib.b2g_route_experts_bwd(None, 64, 1, None, None, None, 0, 1, f(1.0), None, 0, 64, 8, None) == 0
    assert lib.b2g_token_logprobs(None, 8, 0, None, None, 0, None, 0, 8, f(1.0), -100, None, None) == 0
    assert lib.b2g_token_logprobs_bwd(None, 8, 0, None, None, None, 0, None, 8, 0, 8, f(1.0), -100, None) == 0
    assert lib.b2g_policy_loss(None, 8, 0, None, None, None, None, None, f(0.2), f(0.2), f(0), f(1), None, None, None, None, 8, 0, 8, -100, None, None) == 0
    assert lib.b2g_preference_loss(None, 0, None, 0, None, None, 0, 0, -100, f(0.1), f(0), 0, 0, None, None, None, None, None, None) == 0
    assert lib.b2g_preference_loss_bwd(None, None, None, None, None, 0, 0, 0, -100, None) == 0


def test_loss_entries(lib):
    def policy(low=0.2, high=0.2, kl=0.0, tau=1.0, rows=2, v=8, ld=8, ld_out=8, dtype=0):
        rc = lib.b2g_policy_loss(None, ld, dtype, None, None, None, None, None, f(low), f(high), f(kl), f(tau), None, None, None, None, ld_out, rows,
                                 v, -100, None, None)
        return rc, lib.b2g_last_error()

    for kw, what in ((dict(low=1.5), b"clip_low"), (dict(high=-1.0), b"clip_high"), (dict(high=float("nan")), b"clip_high"), (dict(kl=-0.1), b"kl_coef"),
                     (dict(kl=0.1), b"reference"), (dict(tau=0.0), b"temperature"), (dict(tau=float("inf")), b"temperature"),
                     (dict(tau=float("nan")), b"temperature"), (dict(ld=7), b"bad shape"), (dict(ld_out=7), b"bad shape"), (dict(rows=-1), b"bad shape"),
                     (dict(v=0), b"bad shape"), (dict(dtype=2), b"logits_dtype"), (dict(), b"null")):
        rc, msg = policy(**kw)
        assert rc == -1 and what in msg, kw
    assert lib.b2g_token_logprobs(None, 8, 0, None, None, 2, None, 2, 8, f(1.0), -100, None, None) == -1 and b"logp_dtype" in lib.b2g_last_error()

    def pairs(beta=0.1, smooth=0.0, kind=0, pairs_=2, dtype=0):
        rc = lib.b2g_preference_loss(None, dtype, None, 0, None, None, 4, pairs_, -100, f(beta), f(smooth), kind, 0, None, None, None, None, None, None)
        return rc, lib.b2g_last_error()

    for kw, what in ((dict(beta=0.0), b"beta"), (dict(smooth=0.5), b"label_smoothing"), (dict(kind=2), b"loss_type"), (dict(kind=1, smooth=0.1), b"smoothing"),
                     (dict(pairs_=-1), b"bad shape"), (dict(dtype=3), b"logp_dtype"), (dict(), b"null")):
        rc, msg = pairs(**kw)
        assert rc == -1 and what in msg, kw


def test_route_experts_python_refusals():
    from fast_moe_ranking import route_experts

    x = torch.zeros(4, 64)
    for kw, what in ((dict(top_k=0), "top_k"), (dict(top_k=65), "top_k"), (dict(top_k=4, num_groups=7), "groups"),
                     (dict(top_k=4, num_groups=8, top_groups=9), "groups"), (dict(top_k=9, num_groups=8, top_groups=1), "top_k"),
                     (dict(top_k=4, group_experts=3), "group_experts"), (dict(top_k=4, score_function="tanh"), "score function"),
                     (dict(top_k=4, correction_bias=torch.zeros(63)), "correction bias")):
        with pytest.raises(ValueError, match=what):
            route_experts(x, **kw)
    with pytest.raises(ValueError, match="tokens,experts"):
        route_experts(x[0], 4)
    with pytest.raises(ValueError, match="1 to 512"):
        route_experts(torch.zeros(2, 513), 4)
    with pytest.raises(RuntimeError, match="requires CUDA"):
        route_experts(x, 4)


def test_losses_have_no_cpu_path():
    from b2g import ops

    x, t, a = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64), torch.zeros(2)
    for call in (lambda: ops.token_logprobs(x, t), lambda: ops.policy_loss(x, t, a), lambda: ops.preference_loss(a, torch.zeros(3, dtype=torch.int64)),
                 lambda: ops.route_experts(x, 2)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_packed_losses_refuse_other_heads():
    import gguf_policy_loss as gp
    from b2g.gguf_types import GGUFLinear

    head = GGUFLinear(256, 64)
    h, t = torch.zeros(3, 256, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(TypeError, match="GGUFQuantizedTensor"):
        gp.packed_token_logprobs(h, head, t)
    with pytest.raises(TypeError, match="advantages"):
        import unittest.mock as mock
        with mock.patch.object(gp, "_head", return_value=(h, t, t, 8, 64)):
            gp.packed_policy_loss(h, head, t, None)
