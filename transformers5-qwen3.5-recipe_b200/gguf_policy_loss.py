"""Post-training losses on a packed LM head: token log-probabilities, the clipped policy loss and the preference loss.

The supervised loss of ``gguf_liger_loss`` / ``deepseek_v4_liger_loss`` has these next to it: per chunk of hidden-state rows the
packed product makes bf16 logits, a loss kernel turns them into log-probabilities or, in place, into their cotangents, and
the packed input-gradient product takes those back through the head, so that neither a logical LM-head matrix nor the logits of
the whole batch ever exist.  The reference has supervised losses only; names and refusals follow its packed loss
(``gguf_liger_loss.py:263-330``).

``target`` is the token that each row's distribution is asked about (labels already shifted); rows whose target is
``ignore_index`` take no part.
"""
from __future__ import annotations

from typing import Optional

import torch

from b2g import autograd as _ag
from b2g import ops as _ops
from b2g.gguf_types import GGUFQuantizedTensor
from deepseek_v4_liger_loss import _PACKED_LM_HEAD_CHUNK_SIZE


def _head(hidden_states: torch.Tensor, lm_head, target: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, int, int]:
    """(hidden rows, flat targets, payload, quant type, vocabulary) of a packed head that the losses can run on."""
    if not isinstance(lm_head.weight, GGUFQuantizedTensor):
        raise TypeError("Packed LM-head losses require a GGUFQuantizedTensor weight.")
    if lm_head.input_permutation is not None or lm_head.output_permutation is not None:
        raise RuntimeError("Packed LM-head losses do not support layout permutations.")
    if lm_head.compute_dtype != torch.bfloat16:
        raise RuntimeError("Packed LM-head losses require BF16 compute_dtype.")
    if getattr(lm_head, "bias", None) is not None:
        raise RuntimeError("Packed LM-head losses require a bias-free LM head.")
    if lm_head.weight.requires_grad:
        raise RuntimeError("Packed LM-head weights must remain frozen.")
    quant_type = int(lm_head.weight.quant_type)
    if quant_type not in _ops.NATIVE_QUANT_TYPES:
        raise RuntimeError(f"Packed LM-head losses do not support GGML type {quant_type}.")
    if hidden_states.dtype != torch.bfloat16:
        raise TypeError(f"Packed LM-head losses require BF16 hidden states, got {hidden_states.dtype}.")
    if hidden_states.shape[-1] != lm_head.in_features:
        raise ValueError(f"Hidden size {hidden_states.shape[-1]} does not match the LM head ({lm_head.in_features}).")
    if target.dtype != torch.long or target.shape != hidden_states.shape[:-1]:
        raise ValueError(f"Targets must be torch.long with shape {tuple(hidden_states.shape[:-1])}, got {target.dtype} {tuple(target.shape)}.")
    rows = hidden_states.reshape(-1, lm_head.in_features).contiguous()
    return rows, target.reshape(-1).contiguous(), lm_head.weight.as_subclass(torch.Tensor).reshape(-1), quant_type, int(lm_head.out_features)


def _chunks(rows: int, chunk_size: int):
    if chunk_size <= 0:
        raise ValueError(f"Packed LM-head chunk_size must be positive, got {chunk_size}.")
    return [(start, min(start + chunk_size, rows)) for start in range(0, rows, chunk_size)]


class _PackedTokenLogprobs(torch.autograd.Function):
    """The logits of a chunk are made again in the backward pass: two packed products per direction instead of a batch of logits."""

    @staticmethod
    def forward(ctx, rows, payload, target, quant_type, vocab, chunk_size, temperature, ignore_index, dtype):
        logp = torch.empty(rows.shape[0], dtype=dtype, device=rows.device)
        stats = torch.empty(rows.shape[0], 4, dtype=torch.float32, device=rows.device)
        for a, b in _chunks(rows.shape[0], chunk_size):
            logits = torch.ops.b2g.mmq(rows[a:b], payload, quant_type, vocab)
            logp[a:b], stats[a:b] = _ops.token_logprobs(logits, target[a:b], temperature, ignore_index, dtype)
        ctx.save_for_backward(rows, payload, target, stats)
        ctx.settings = (quant_type, vocab, chunk_size, temperature, ignore_index)
        return logp

    @staticmethod
    def backward(ctx, grad_logp):
        if torch.is_grad_enabled():
            raise RuntimeError("Packed LM-head losses do not support higher-order gradients")
        rows, payload, target, stats = ctx.saved_tensors
        quant_type, vocab, chunk_size, temperature, ignore_index = ctx.settings
        grad_logp = grad_logp.contiguous()
        grad = torch.empty_like(rows)
        for a, b in _chunks(rows.shape[0], chunk_size):
            logits = torch.ops.b2g.mmq(rows[a:b], payload, quant_type, vocab)
            _ops.token_logprobs_bwd(grad_logp[a:b], logits, target[a:b], stats[a:b], temperature, ignore_index, out=logits)
            grad[a:b] = torch.ops.b2g.mmq_grad_input(logits, payload, quant_type, rows.shape[1])
        return (grad,) + (None,) * 8


class _PackedPolicyLoss(torch.autograd.Function):
    """The input gradient is finished in the forward pass and only scaled in the backward pass."""

    @staticmethod
    def forward(ctx, rows, payload, target, advantage, old_logp, ref_logp, weight, quant_type, vocab, chunk_size, settings):
        n = rows.shape[0]
        wanted = ctx.needs_input_grad[0]
        loss, logp, kl = (torch.empty(n, dtype=torch.float32, device=rows.device) for _ in range(3))
        grad = torch.empty_like(rows) if wanted else None

        def part(t, a, b):
            return None if t is None else t[a:b]

        for a, b in _chunks(n, chunk_size):
            logits = torch.ops.b2g.mmq(rows[a:b], payload, quant_type, vocab)
            loss[a:b], logp[a:b], kl[a:b], _ = _ops.policy_loss(logits, target[a:b], advantage[a:b], old_logp=part(old_logp, a, b),
                                                                ref_logp=part(ref_logp, a, b), weight=part(weight, a, b), out=logits, **settings)
            if wanted:
                grad[a:b] = torch.ops.b2g.mmq_grad_input(logits, payload, quant_type, rows.shape[1])
        if wanted:
            ctx.save_for_backward(grad)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(logp, kl)
        return loss.sum(), logp, kl

    @staticmethod
    def backward(ctx, grad_loss, _grad_logp, _grad_kl):
        if torch.is_grad_enabled():
            raise RuntimeError("Packed LM-head losses do not support higher-order gradients")
        if grad_loss is None:
            return (None,) * 11
        (grad,) = ctx.saved_tensors
        return (grad.float().mul_(grad_loss).to(grad.dtype),) + (None,) * 10      # a bf16 factor would be off by 2^-9 everywhere


def packed_token_logprobs(hidden_states: torch.Tensor, lm_head, target: torch.Tensor, *, temperature: float = 1.0, ignore_index: int = -100,
                          dtype: torch.dtype = torch.float32, chunk_size: int = _PACKED_LM_HEAD_CHUNK_SIZE) -> torch.Tensor:
    """Log-probabilities (fp32 or fp64, shaped like ``target``) of the target tokens, 0 where the target is ``ignore_index``;
    they carry the gradient to the hidden states.  Under ``torch.no_grad`` this scores a batch for the old or the reference policy."""
    rows, flat, payload, quant_type, vocab = _head(hidden_states, lm_head, target)
    logp = _PackedTokenLogprobs.apply(rows, payload, flat, quant_type, vocab, int(chunk_size), float(temperature), int(ignore_index), dtype)
    return logp.reshape(target.shape)


def packed_policy_loss(hidden_states: torch.Tensor, lm_head, target: torch.Tensor, advantage: torch.Tensor, *,
                       old_logp: Optional[torch.Tensor] = None, ref_logp: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                       clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0, temperature: float = 1.0, ignore_index: int = -100,
                       chunk_size: int = _PACKED_LM_HEAD_CHUNK_SIZE) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(loss, logp, kl)``: the sum over tokens of ``ops.policy_loss`` on the packed head, with the gradient of the hidden
    states, and the tokens' log-probabilities and KL estimates for logging.  ``weight`` carries the normalisation (one over the
    token count, or over the answer's length and the number of answers).  All per-token tensors are fp32 and shaped like ``target``."""
    rows, flat, payload, quant_type, vocab = _head(hidden_states, lm_head, target)
    if advantage is None:
        raise TypeError("packed_policy_loss needs advantages")
    per_token = []
    for name, t in (("advantage", advantage), ("old_logp", old_logp), ("ref_logp", ref_logp), ("weight", weight)):
        if t is not None and (t.shape != target.shape or t.dtype != torch.float32):
            raise ValueError(f"{name} must be fp32 with shape {tuple(target.shape)}, got {t.dtype} {tuple(t.shape)}")
        per_token.append(None if t is None else t.detach().reshape(-1).contiguous())
    if not torch.is_grad_enabled():
        rows = rows.detach()                  # nobody will ask for the input gradient
    settings = dict(clip_low=clip_low, clip_high=clip_high, kl_coef=kl_coef, temperature=temperature, ignore_index=ignore_index)
    loss, logp, kl = _PackedPolicyLoss.apply(rows, payload, flat, *per_token, quant_type, vocab, int(chunk_size), settings)
    return loss, logp.reshape(target.shape), kl.reshape(target.shape)


def packed_preference_loss(hidden_states: torch.Tensor, lm_head, target: torch.Tensor, offsets: torch.Tensor, *,
                           ref_logp: Optional[torch.Tensor] = None, beta: float = 0.1, label_smoothing: float = 0.0, loss_type: str = "sigmoid",
                           average: bool = False, ignore_index: int = -100,
                           chunk_size: int = _PACKED_LM_HEAD_CHUNK_SIZE) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(loss [pairs], chosen rewards, rejected rewards)`` of ``ops.preference_loss`` on the packed head.  The tokens of all
    sequences lie one behind the other (``hidden_states [tokens, hidden]``), the chosen sequences first; ``offsets`` has
    ``2 * pairs + 1`` entries.  A target outside the vocabulary is reported through the status word (902) and takes no part, in the
    sums and in the mean's count alike."""
    if target.dim() != 1:
        raise ValueError(f"packed_preference_loss takes the sequences one behind the other, got targets {tuple(target.shape)}")
    logp = packed_token_logprobs(hidden_states, lm_head, target, ignore_index=ignore_index, dtype=torch.float64, chunk_size=chunk_size)
    # the pairs' kernel knows no vocabulary: it is told which tokens the log-probabilities have left out
    target = target.masked_fill((target < 0) | (target >= int(lm_head.out_features)), ignore_index)
    return _ag.preference_loss(logp, offsets, ref_logp, beta, label_smoothing, loss_type, average, target, ignore_index)
