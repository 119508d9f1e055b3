"""CPU restatement of expert routing and the post-training losses in 64 bits, from their formulas."""
from __future__ import annotations

import math

import torch


def scores(logits: torch.Tensor, fn: str) -> torch.Tensor:
    x = logits.double()
    if fn == "sigmoid":
        return torch.sigmoid(x)
    if fn == "sqrtsoftplus":
        return torch.sqrt(x.clamp(min=0) + torch.log1p(torch.exp(-x.abs())))
    top = x.amax(1, keepdim=True)
    e = torch.where(torch.isneginf(top), torch.zeros_like(x), torch.exp(x - top))
    total = e.sum(1, keepdim=True)
    return torch.where(total > 0, e / total.clamp(min=1e-300), torch.zeros_like(e))


def choose(logits: torch.Tensor, top_k: int, bias=None, fn: str = "softmax", groups: int = 1, top_groups: int = 1, group_experts: int = 1) -> torch.Tensor:
    """Expert ids by brute force: sorted by (choice descending, id ascending) among the experts of the kept groups."""
    s = scores(logits, fn)
    choice = logits.double() if bias is None else s + bias.double()
    value = s if bias is None else choice
    t, e = choice.shape
    per = e // groups
    out = torch.empty(t, top_k, dtype=torch.int64)
    for r in range(t):
        c, v = choice[r].tolist(), value[r].tolist()
        worth = [sum(sorted(v[g * per:(g + 1) * per], reverse=True)[:group_experts]) for g in range(groups)]
        kept = set(sorted(range(groups), key=lambda g: (-worth[g], g))[:top_groups])
        ids = sorted((i for i in range(e) if i // per in kept), key=lambda i: (-c[i], i))
        out[r] = torch.tensor(ids[:top_k])
    return out


def weights(logits: torch.Tensor, idx: torch.Tensor, fn: str = "softmax", renormalize: bool = True, alpha: float = 1.0) -> torch.Tensor:
    """Differentiable in ``logits`` (float64)."""
    if renormalize and fn == "softmax":
        return alpha * torch.softmax(logits.gather(1, idx), 1)
    if fn == "softmax":
        s = torch.softmax(logits, 1)
    elif fn == "sigmoid":
        s = torch.sigmoid(logits)
    else:
        s = torch.sqrt(torch.nn.functional.softplus(logits, threshold=1e9))
    w = s.gather(1, idx)
    return alpha * (w / (w.sum(1, keepdim=True) + 1e-20) if renormalize else w)


def logprobs(logits: torch.Tensor, target: torch.Tensor, tau: float = 1.0, ignore_index: int = -100) -> torch.Tensor:
    """Differentiable in ``logits`` (float64); 0 for ignored rows."""
    live = target != ignore_index
    z = torch.where(live[:, None], logits, torch.zeros_like(logits)) / tau
    return torch.where(live, torch.log_softmax(z, 1).gather(1, target.clamp(min=0)[:, None])[:, 0], torch.zeros((), dtype=torch.float64))


def policy(logp, advantage, old=None, ref=None, weight=None, low=0.2, high=0.2, kl_coef=0.0, live=None):
    """(loss, kl, d loss / d logp) per token, the derivative from its formula."""
    a = advantage.double()
    r = torch.exp(logp - old.double()) if old is not None else torch.ones_like(logp)
    clipped = r.clamp(1 - low, 1 + high)
    inside = r * a <= clipped * a
    loss, slope = -torch.minimum(r * a, clipped * a), torch.where(inside, -r * a, torch.zeros_like(a))
    kl = torch.zeros_like(logp)
    if ref is not None:
        d = ref.double() - logp
        kl = torch.expm1(d) - d
        loss, slope = loss + kl_coef * kl, slope - kl_coef * torch.expm1(d)
    w = torch.ones_like(a) if weight is None else weight.double()
    zero = torch.zeros_like(a)
    on = (w != 0) if live is None else live & (w != 0)
    return torch.where(on, w * loss, zero), torch.where(on, kl, zero), torch.where(on, w * slope, zero)


def preference(logp, offsets, ref=None, beta=0.1, smoothing=0.0, kind="sigmoid", average=False, target=None, ignore_index=-100):
    """(loss, chosen, rejected) of pairs; differentiable in ``logp`` (float64)."""
    ends = offsets.tolist()
    value = []
    for a, b in zip(ends[:-1], ends[1:]):
        keep = torch.ones(b - a, dtype=torch.bool) if target is None else target[a:b] != ignore_index
        part = logp[a:b][keep] - (ref[a:b][keep].double() if ref is not None else 0.0)
        value.append(part.sum() / (max(1, int(keep.sum())) if average else 1))
    value = torch.stack(value) if value else logp.new_zeros(0)
    pairs = len(value) // 2
    gap = value[:pairs] - value[pairs:]
    if kind == "sigmoid":
        ls = torch.nn.functional.logsigmoid
        loss = -(1 - smoothing) * ls(beta * gap) - smoothing * ls(-beta * gap)
    else:
        loss = (gap - 0.5 / beta) ** 2
    return loss, beta * value[:pairs], beta * value[pairs:]


# Half a step relative to a value, and the error that the kernels' 32-bit arithmetic can add.
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def lse_error(vocab: int) -> float:
    """Largest error of a row's log-sum-exp.  A term carries at most 2^-22 (the exponential), 3 * 2^-24 (a tree of eight terms)
    and 2 * 2^-24 of its exponent t (product and fma); weighted by the terms, |t| is at most log2(vocab) on average."""
    return 2.0 ** -22 + 2.0 ** -24 * (3 + 2 * math.log(max(vocab, 2)))
