"""CPU: what the autograd surfaces of routing and losses cannot differentiate they refuse, whatever kind of derivative was asked for.

The kernels are replaced by functions that return tensors of the right shapes: only the way to them is looked at."""
from unittest import mock

import pytest
import torch
from torch.autograd import forward_ad as fwad


def _route(logits, top_k, *_):
    return torch.zeros(logits.shape[0], top_k), torch.zeros(logits.shape[0], top_k, dtype=torch.int64)


def _logp(logits, target, *_):
    return torch.zeros(logits.shape[0]), torch.zeros(logits.shape[0], 4)


def _pairs(logp, offsets, *_):
    pairs = offsets.numel() // 2
    return torch.zeros(pairs), torch.zeros(pairs), torch.zeros(pairs), torch.zeros(2 * pairs)


def _calls():
    from b2g import autograd as ag

    t, ends = torch.zeros(3, dtype=torch.int64), torch.tensor([0, 1, 3])
    return [lambda x: ag.route_experts(x, 2)[0], lambda x: ag.token_logprobs(x, t), lambda x: ag.preference_loss(x[:, 0], ends)[0]]


@pytest.fixture()
def surfaces():
    from b2g import ops

    with mock.patch.object(ops, "route_experts", _route), mock.patch.object(ops, "token_logprobs", _logp), mock.patch.object(ops, "preference_loss", _pairs):
        yield _calls()


def test_a_forward_mode_tangent_is_not_dropped(surfaces):
    for call in surfaces:
        with fwad.dual_level():
            dual = fwad.make_dual(torch.zeros(3, 8), torch.ones(3, 8))
            with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward"):
                call(dual)
            # a tensor without a tangent is an ordinary one, also inside such a level
            assert fwad.unpack_dual(call(torch.zeros(3, 8))).tangent is None
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward"):
            with fwad.dual_level():
                call(fwad.make_dual(torch.zeros(3, 8, requires_grad=True), torch.ones(3, 8)))


def test_without_a_gradient_to_carry_there_is_no_node(surfaces):
    for call in surfaces:
        assert call(torch.zeros(3, 8)).grad_fn is None
        with torch.no_grad():
            assert call(torch.zeros(3, 8, requires_grad=True)).grad_fn is None
        assert call(torch.zeros(3, 8, requires_grad=True)).grad_fn is not None
