"""Cases that time the post-training operators: routing to experts, token log-probabilities, the clipped policy loss and
the preference loss.

Every case has a plain form in elementary torch operations, the call of the framework's own operator (``own``), and the
definition in 64 bits (``exact``).  Vocabulary widths 248320 and 129280, 256 experts and top 8 / top 6 are those of the
framework's configurations; the other sizes are generic.
"""
import math
import os
import sys

import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "transformers5-qwen3.5-recipe_b200")
_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_IGNORE = -100


# --------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------
def _route(name, tokens, experts, top_k, dtype, score, bias, groups=1, kept=1, best=1, renorm=True, scale=1.0, backward=True):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype, "score": score, "bias": bias,
            "groups": groups, "kept": kept, "best": best, "renorm": renorm, "scale": scale, "backward": backward}


def _logp(name, rows, vocab, dtype, temperature=1.0, backward=True):
    return {"name": name, "op": "logp", "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": temperature, "backward": backward}


def _policy(name, rows, vocab, dtype, temperature=1.0, kl=0.04, low=0.2, high=0.2, old=True):
    return {"name": name, "op": "policy", "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": temperature, "kl": kl, "low": low,
            "high": high, "old": old}


def _pairs(name, pairs, length, loss, vocab=0, dtype="bf16", beta=0.1, smoothing=0.0, average=False, ref=True):
    return {"name": name, "op": "pairs", "pairs": pairs, "length": length, "loss": loss, "vocab": vocab, "dtype": dtype, "beta": beta,
            "smoothing": smoothing, "average": average, "ref": ref}


def listed():
    return [
        # one decoded token through a layer's router: latency only
        _route("route one token", 1, 256, 8, "bf16", "softmax", False, backward=False),
        # a decode batch with a balance bias
        _route("route decode batch", 96, 256, 6, "fp32", "sqrtsoftplus", True, scale=1.5, backward=False),
        # a training micro-batch, grouped routing (8 groups, 4 kept by their two best)
        _route("route groups train", 8192, 256, 8, "fp32", "sigmoid", True, 8, 4, 2, True, 2.5),
        # the largest token count of the framework's routing path
        _route("route 64k train", 65536, 256, 8, "bf16", "softmax", False),
        # a width that is no power of two, weights not renormalised (the gradient reaches every expert), odd token count
        _route("route odd", 1237, 96, 5, "fp32", "softmax", False, 1, 1, 1, False, 1.0),
        # scoring a stored batch under the old policy: forward only
        _logp("logp score", 1024, 248320, "bf16", backward=False),
        # a short answer, forward and backward
        _logp("logp short", 23, 129280, "bf16"),
        # one token of a policy update: the smallest work of the loss
        _policy("policy one token", 1, 248320, "bf16"),
        # the chunk of a packed head
        _policy("policy chunk", 1024, 248320, "bf16"),
        # fp32 logits of a small odd vocabulary, a temperature, asymmetric clipping
        _policy("policy odd", 301, 32003, "fp32", 0.7, 0.1, 0.2, 0.28),
        # chosen / rejected answers from logits to the gradient of the logits
        _pairs("pairs from logits", 4, 128, "sigmoid", 129280),
        # stored log-probabilities of many ragged answers
        _pairs("pairs long", 64, 8192, "squared", average=True),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, uniform in its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["route", "route", "logp", "policy", "policy", "pairs"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        per = _spread(rng, 2, 512 // groups)
        experts = groups * per
        kept = rng.randint(1, groups)
        top_k = rng.randint(1, min(16, kept * per))
        tokens = _spread(rng, 1, 65536 * 256 // max(256, experts))
        case = _route("", tokens, experts, top_k, dtype, rng.choice(["softmax", "sigmoid", "sqrtsoftplus"]), rng.random() < 0.5, groups, kept,
                      rng.choice([1, 2]), rng.random() < 0.75, rng.choice([1.0, 1.5, 2.5]), rng.random() < 0.7)
    else:
        vocab = _spread(rng, 1000, 248320)
        if rng.random() < 0.5:
            vocab = max(1000, vocab // 64 * 64)
        size = 2 if dtype == "bf16" else 4
        rows = _spread(rng, 1, max(1, min(16384, 1024 * 248320 * 2 // (vocab * size))))
        if op == "logp":
            case = _logp("", rows, vocab, dtype, rng.choice([1.0, 1.0, 0.8]), rng.random() < 0.6)
        elif op == "policy":
            case = _policy("", rows, vocab, dtype, rng.choice([1.0, 1.0, 0.9]), rng.choice([0.0, 0.01, 0.1]), 0.2, rng.choice([0.2, 0.28]),
                           rng.random() < 0.8)
        else:
            pairs = _spread(rng, 1, 256)
            kind = rng.choice(["sigmoid", "squared"])
            smoothing = rng.choice([0.0, 0.1]) if kind == "sigmoid" else 0.0
            if rng.random() < 0.4:
                length = max(1, min(1024, rows // (4 * pairs)))
                case = _pairs("", pairs, length, kind, min(vocab, 1024 * 248320 // (4 * pairs * length)), dtype, rng.choice([0.05, 0.1, 0.5]),
                              smoothing, rng.random() < 0.5, True)
            else:
                length = _spread(rng, 1, min(32768, 2 * 1024 * 1024 // pairs))
                case = _pairs("", pairs, length, kind, 0, "fp32", rng.choice([0.05, 0.1, 0.5]), smoothing, rng.random() < 0.5,
                              rng.random() < 0.8)
    del case["name"]
    return case


# --------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------
def _logit_rows(gen, rows, vocab, dtype):
    """Head outputs of a trained model: a spread of a few units, and one token that stands out by an amount of its own."""
    logits = torch.randn(rows, vocab, generator=gen, device="cuda", dtype=torch.float32).mul_(2.0)
    target = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    lift = 6.0 + 10.0 * torch.rand(rows, generator=gen, device="cuda")
    logits[torch.arange(rows, device="cuda"), target] = lift
    return logits.to(dtype), target


def _true_logp(logits, target, temperature):
    out = []
    for z, y in zip(logits.split(128), target.split(128)):
        z = z.float() / temperature
        out.append(z.gather(1, y[:, None])[:, 0] - torch.logsumexp(z, dim=1))
    return torch.cat(out)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"

    def normal(n, scale):
        return torch.randn(n, generator=gen, device=dev) * scale

    state = {"case": case}
    if case["op"] == "route":
        t, e = case["tokens"], case["experts"]
        logits = torch.randn(t, e, generator=gen, device=dev).mul_(1.5).to(_DTYPES[case["dtype"]])
        state["logits"] = logits.requires_grad_(case["backward"])
        state["bias"] = normal(e, 0.05) if case["bias"] else None
        state["grad"] = torch.randn(t, case["top_k"], generator=gen, device=dev) if case["backward"] else None
        return state
    if case["op"] in ("logp", "policy"):
        rows, tau = case["rows"], case["temperature"]
        logits, target = _logit_rows(gen, rows, case["vocab"], _DTYPES[case["dtype"]])
        logp = _true_logp(logits, target, tau)
        if rows > 8:   # prompt and padding tokens take no part
            target[torch.rand(rows, generator=gen, device=dev) < 0.1] = _IGNORE
        state["target"] = target
        if case["op"] == "logp":
            state["logits"] = logits.requires_grad_(case["backward"])
            state["grad"] = normal(rows, 1.0 / rows) if case["backward"] else None
            return state
        state["logits"] = logits
        state["old"] = logp + normal(rows, 0.1) if case["old"] else None
        state["ref"] = logp + normal(rows, 0.2) if case["kl"] > 0 else None
        state["advantage"] = normal(rows, 1.0)
        state["weight"] = torch.full((rows,), 1.0 / rows, device=dev)
        return state
    # answers of ragged lengths (one in sixteen is empty), the chosen ones first
    count = 2 * case["pairs"]
    lengths = (torch.rand(count, generator=gen, device=dev) * (case["length"] + 1)).long().clamp(max=case["length"])
    if count > 4:
        lengths[torch.rand(count, generator=gen, device=dev) < 1 / 16] = 0
    # the token rows are as many as the longest batch could hold: the tail behind the last answer belongs to nobody
    rows = max(1, count * case["length"])
    state["offsets"] = torch.cat([lengths.new_zeros(1), lengths.cumsum(0)])
    if case["vocab"]:
        logits, target = _logit_rows(gen, rows, case["vocab"], _DTYPES[case["dtype"]])
        logp = _true_logp(logits, target, 1.0)
        state["logits"] = logits.requires_grad_(True)
    else:
        logp = -torch.rand(rows, generator=gen, device=dev).pow_(4).mul_(8.0)
        target = torch.zeros(rows, dtype=torch.long, device=dev)
        state["logp"] = logp.requires_grad_(True)
    target[torch.rand(rows, generator=gen, device=dev) < 0.05] = _IGNORE
    state["target"] = target
    state["ref"] = logp.detach() + normal(rows, 0.05) if case["ref"] else None
    state["grad"] = torch.full((case["pairs"],), 1.0 / case["pairs"], device=dev)
    return state


# --------------------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------------------
def _plain_route(s):
    c = s["case"]
    t, e, k, alpha = c["tokens"], c["experts"], c["top_k"], c["scale"]
    raw = s["logits"].detach()
    x = raw.double()      # choices that lie close together keep their order
    if c["score"] == "softmax":
        score = torch.exp(x - x.amax(1, keepdim=True))
        score = score / score.sum(1, keepdim=True)
    elif c["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-x))
    else:
        score = torch.sqrt(torch.clamp(x, min=0) + torch.log1p(torch.exp(-torch.abs(x))))
    choice = x if s["bias"] is None else score + s["bias"].double()
    if c["groups"] > 1:
        value = score if s["bias"] is None else choice
        best = value.view(t, c["groups"], -1).sort(dim=2, descending=True).values[:, :, :c["best"]].sum(2)
        keep = best.sort(dim=1, descending=True, stable=True).indices[:, :c["kept"]]
        mask = torch.zeros(t, c["groups"], dtype=torch.bool, device=x.device)
        mask[torch.arange(t, device=x.device)[:, None], keep] = True
        choice = torch.where(mask.repeat_interleave(e // c["groups"], 1), choice, torch.full_like(choice, -math.inf))
    idx = choice.sort(dim=1, descending=True, stable=True).indices[:, :k]
    chosen = score[torch.arange(t, device=x.device)[:, None], idx]
    total = chosen.sum(1, keepdim=True) + 1e-20
    w = alpha * chosen / total if c["renorm"] else alpha * chosen
    if not c["backward"]:
        return w.float(), idx
    g = s["grad"].double()
    ds = (alpha * g - (g * w).sum(1, keepdim=True)) / total if c["renorm"] else alpha * g
    rows = torch.arange(t, device=x.device)[:, None]
    if c["score"] == "softmax":
        full = torch.zeros_like(score)
        full[rows, idx] = ds
        grad = score * (full - (ds * chosen).sum(1, keepdim=True))
    else:
        sig = 1.0 / (1.0 + torch.exp(-x[rows, idx]))
        rest = 1.0 / (1.0 + torch.exp(x[rows, idx]))
        slope = sig * rest if c["score"] == "sigmoid" else sig / (2.0 * chosen)
        grad = torch.zeros_like(score)
        grad[rows, idx] = ds * slope
    return w.float(), idx, grad.to(raw.dtype)


def _plain_rows(logits, target, temperature):
    """Scaled logits in 32 bits, their log-sum-exp, the targets' log-probabilities and who takes part."""
    z = logits.detach().float()
    if temperature != 1.0:
        z = z / temperature
    top = z.amax(1)
    lse = top.double() + torch.log(torch.exp(z - top[:, None]).sum(1, dtype=torch.float64))
    live = target != _IGNORE
    y = torch.where(live, target, torch.zeros_like(target))
    logp = z[torch.arange(z.shape[0], device=z.device), y].double() - lse
    return z, lse, torch.where(live, logp, torch.zeros_like(logp)), live, y


def _plain_cotangent(z, lse, live, y, coefficient, dtype):
    """coefficient * (onehot - softmax), zero where a row takes no part."""
    grad = torch.exp(z - lse.float()[:, None]).neg_()
    grad[torch.arange(z.shape[0], device=z.device), y] += 1.0
    grad *= torch.where(live, coefficient, torch.zeros_like(coefficient)).float()[:, None]
    return grad.to(dtype)


def _plain_logp(s):
    c = s["case"]
    z, lse, logp, live, y = _plain_rows(s["logits"], s["target"], c["temperature"])
    if not c["backward"]:
        return logp.float()
    return logp.float(), _plain_cotangent(z, lse, live, y, s["grad"].double() / c["temperature"], s["logits"].dtype)


def _plain_policy(s):
    c = s["case"]
    z, lse, logp, live, y = _plain_rows(s["logits"], s["target"], c["temperature"])
    a, w = s["advantage"].double(), s["weight"].double()
    ratio = torch.exp(logp - s["old"].double()) if s["old"] is not None else torch.ones_like(logp)
    clipped = torch.clamp(ratio, 1.0 - c["low"], 1.0 + c["high"])
    loss = -torch.minimum(ratio * a, clipped * a)
    slope = torch.where(ratio * a <= clipped * a, -a * ratio, torch.zeros_like(a))
    kl = torch.zeros_like(logp)
    if s["ref"] is not None:
        d = s["ref"].double() - logp
        kl = torch.exp(d) - d - 1.0
        loss = loss + c["kl"] * kl
        slope = slope + c["kl"] * (1.0 - torch.exp(d))
    zero = torch.zeros_like(loss)
    grad = _plain_cotangent(z, lse, live, y, w * slope / c["temperature"], s["logits"].dtype)
    return torch.where(live, w * loss, zero).float(), logp.float(), torch.where(live, kl, zero).float(), grad


def _plain_pair_loss(c, logp, ref, target, offsets, g):
    """Loss and rewards of every pair, and the gradient of every token's log-probability."""
    rows, pairs, beta = logp.shape[0], c["pairs"], c["beta"]
    place = torch.arange(rows, device=logp.device)
    seq = (place[:, None] >= offsets[None, 1:]).sum(1) if rows * offsets.numel() < 1 << 28 else torch.bucketize(place, offsets[1:], right=True)
    counted = (seq < 2 * pairs) & (target != _IGNORE)
    diff = logp.double() - (ref.double() if ref is not None else 0.0)
    diff = torch.where(counted, diff, torch.zeros_like(diff))
    seq = torch.where(counted, seq, torch.zeros_like(seq))
    total = torch.zeros(2 * pairs, dtype=torch.float64, device=logp.device).index_add_(0, seq, diff)
    count = torch.ones_like(total)
    if c["average"]:
        count = torch.zeros_like(total).index_add_(0, seq, counted.double()).clamp(min=1.0)
        total = total / count
    chosen, rejected = beta * total[:pairs], beta * total[pairs:]
    u = chosen - rejected

    def log_sigmoid(v):
        return torch.clamp(v, max=0) - torch.log1p(torch.exp(-torch.abs(v)))

    if c["loss"] == "sigmoid":
        eps = c["smoothing"]
        loss = -(1.0 - eps) * log_sigmoid(u) - eps * log_sigmoid(-u)
        slope = -(1.0 - eps) / (1.0 + torch.exp(u)) + eps / (1.0 + torch.exp(-u))
    else:
        gap = u / beta - 1.0 / (2.0 * beta)
        loss, slope = gap * gap, 2.0 * gap / beta
    per = g.double() * slope * beta
    per = torch.cat([per, -per]) / count
    grad = torch.where(counted, per[seq], torch.zeros_like(diff))
    return loss.float(), chosen.float(), rejected.float(), grad


def _plain_pairs(s):
    c = s["case"]
    if not c["vocab"]:
        loss, chosen, rejected, grad = _plain_pair_loss(c, s["logp"].detach(), s["ref"], s["target"], s["offsets"], s["grad"])
        return loss, chosen, rejected, grad.float()
    z, lse, logp, live, y = _plain_rows(s["logits"], s["target"], 1.0)
    loss, chosen, rejected, g = _plain_pair_loss(c, logp, s["ref"], s["target"], s["offsets"], s["grad"])
    return loss, chosen, rejected, logp.float(), _plain_cotangent(z, lse, live, y, g, s["logits"].dtype)


# --------------------------------------------------------------------------------------
# the framework's operators
# --------------------------------------------------------------------------------------
def _own(s):
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from b2g import autograd, ops
    from fast_moe_ranking import route_experts

    c = s["case"]
    if c["op"] == "route":
        w, idx = route_experts(s["logits"], c["top_k"], correction_bias=s["bias"], score_function=c["score"], num_groups=c["groups"],
                               top_groups=c["kept"], group_experts=c["best"], renormalize=c["renorm"], scaling_factor=c["scale"])
        if not c["backward"]:
            return w, idx
        return w.detach(), idx, torch.autograd.grad(w, s["logits"], s["grad"])[0]
    if c["op"] == "logp":
        logp = autograd.token_logprobs(s["logits"], s["target"], temperature=c["temperature"], ignore_index=_IGNORE)
        if not c["backward"]:
            return logp
        return logp.detach(), torch.autograd.grad(logp, s["logits"], s["grad"])[0]
    if c["op"] == "policy":
        return ops.policy_loss(s["logits"], s["target"], s["advantage"], old_logp=s["old"], ref_logp=s["ref"], weight=s["weight"],
                               clip_low=c["low"], clip_high=c["high"], kl_coef=c["kl"], temperature=c["temperature"], ignore_index=_IGNORE)
    settings = dict(beta=c["beta"], label_smoothing=c["smoothing"], loss_type=c["loss"], average=c["average"], target=s["target"],
                    ignore_index=_IGNORE)
    if not c["vocab"]:
        loss, chosen, rejected = autograd.preference_loss(s["logp"], s["offsets"], ref_logp=s["ref"], **settings)
        return loss.detach(), chosen, rejected, torch.autograd.grad(loss, s["logp"], s["grad"])[0]
    # the sequences' sums of differences need more digits of the log-probabilities than 32 bits hold
    logp = autograd.token_logprobs(s["logits"], s["target"], ignore_index=_IGNORE, dtype=torch.float64)
    loss, chosen, rejected = autograd.preference_loss(logp, s["offsets"], ref_logp=s["ref"], **settings)
    return loss.detach(), chosen, rejected, logp.detach().float(), torch.autograd.grad(loss, s["logits"], s["grad"])[0]


def run(state):
    if own:
        return _own(state)
    return {"route": _plain_route, "logp": _plain_logp, "policy": _plain_policy, "pairs": _plain_pairs}[state["case"]["op"]](state)


# --------------------------------------------------------------------------------------
# bytes and operations that a pass cannot do without
# --------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        size = 2 if case["dtype"] == "bf16" else 4
        total = t * e * size + t * k * 12 + (4 * e if case["bias"] else 0)
        if case["backward"]:
            total += t * k * 4 + t * e * size
        return {"bytes": total, "flops": t * e * (12 if case["backward"] else 8)}
    if case["op"] in ("logp", "policy"):
        n, v = case["rows"], case["vocab"]
        size = 2 if case["dtype"] == "bf16" else 4
        both = case["op"] == "policy" or case["backward"]
        row = 8 + 4 + (4 if case["op"] == "logp" and both else 0)
        if case["op"] == "policy":
            row += 4 + 4 + 4 + 4 + (4 if case["old"] else 0) + (4 if case["kl"] > 0 else 0)
        return {"bytes": n * v * size * (2 if both else 1) + n * row, "flops": n * v * (8 if both else 4)}
    # as many tokens as the batch holds on average; every row has its place in the gradient
    pairs, length = case["pairs"], case["length"]
    rows = max(1, 2 * pairs * length)
    token = 8 + (8 if case["ref"] else 4)
    if not case["vocab"]:
        return {"bytes": int(rows * 0.5 * token) + rows * 4 + pairs * 12, "flops": rows * 4}
    size = 2 if case["dtype"] == "bf16" else 4
    return {"bytes": 2 * rows * case["vocab"] * size + rows * 16 + pairs * 12, "flops": rows * case["vocab"] * 8}


# --------------------------------------------------------------------------------------
# the definition in 64 bits
# --------------------------------------------------------------------------------------
def _exact_route(s):
    c = s["case"]
    x = s["logits"].detach().double().requires_grad_(True)
    if c["score"] == "softmax":
        score = torch.softmax(x, 1)
    elif c["score"] == "sigmoid":
        score = torch.sigmoid(x)
    else:
        score = torch.nn.functional.softplus(x, threshold=1e9).sqrt()
    with torch.no_grad():
        order = x.detach().clone() if s["bias"] is None else score + s["bias"].double()
        if c["groups"] > 1:
            per = c["experts"] // c["groups"]
            value = score if s["bias"] is None else order
            worth = value.view(-1, c["groups"], per).topk(min(c["best"], per), dim=2).values.sum(2)
            for _ in range(c["groups"] - c["kept"]):      # drop the worst group; among equals the last one
                low = worth.amin(1, keepdim=True)
                last = (worth == low).long() * torch.arange(1, c["groups"] + 1, device=x.device)
                drop = last.argmax(1)
                worth[torch.arange(len(worth), device=x.device), drop] = math.inf
                order.view(-1, c["groups"], per)[torch.arange(len(worth), device=x.device), drop] = -math.inf
        picks = []
        ids = torch.arange(c["experts"], device=x.device)
        for _ in range(c["top_k"]):
            top = order.amax(1, keepdim=True)
            pick = torch.where(order == top, ids, c["experts"]).amin(1)
            picks.append(pick)
            order[torch.arange(len(order), device=x.device), pick] = -math.inf
        idx = torch.stack(picks, 1)
    w = score.gather(1, idx)
    if c["renorm"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    w = w * c["scale"]
    if not c["backward"]:
        return w.detach(), idx
    return w.detach(), idx, torch.autograd.grad(w, x, s["grad"].double())[0]


def _exact_logp(logits, target, temperature):
    """log-probabilities (differentiable) and the leaf they are a function of."""
    x = logits.detach().double().requires_grad_(True)
    live = target != _IGNORE
    picked = (x / temperature).gather(1, target.clamp(min=0)[:, None])[:, 0] - torch.logsumexp(x / temperature, 1)
    return x, torch.where(live, picked, 0.0), live


def _exact_pairs(c, logp, ref, target, offsets):
    ends = offsets.tolist()
    live = target != _IGNORE
    value = []
    for begin, end in zip(ends[:-1], ends[1:]):
        keep = live[begin:end]
        part = logp[begin:end][keep]
        if ref is not None:
            part = part - ref[begin:end][keep].double()
        total = part.sum()
        value.append(total / max(1, part.numel()) if c["average"] else total)
    value = torch.stack(value)
    chosen, rejected = c["beta"] * value[:c["pairs"]], c["beta"] * value[c["pairs"]:]
    u = chosen - rejected
    if c["loss"] == "sigmoid":
        logsig = torch.nn.functional.logsigmoid
        loss = -(1 - c["smoothing"]) * logsig(u) - c["smoothing"] * logsig(-u)
    else:
        loss = (u / c["beta"] - 0.5 / c["beta"]) ** 2
    return loss, chosen.detach(), rejected.detach()


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "route":
        return _exact_route(s)
    if c["op"] == "logp":
        x, logp, _ = _exact_logp(s["logits"], s["target"], c["temperature"])
        if not c["backward"]:
            return logp.detach()
        return logp.detach(), torch.autograd.grad(logp, x, s["grad"].double())[0]
    if c["op"] == "policy":
        x, logp, live = _exact_logp(s["logits"], s["target"], c["temperature"])
        a = s["advantage"].double()
        ratio = torch.exp(logp - s["old"].double()) if s["old"] is not None else torch.exp(logp - logp.detach())
        loss = -torch.minimum(ratio * a, ratio.clamp(1 - c["low"], 1 + c["high"]) * a)
        kl = torch.zeros_like(logp)
        if s["ref"] is not None:
            d = s["ref"].double() - logp
            kl = torch.expm1(d) - d
            loss = loss + c["kl"] * kl
        loss = torch.where(live, s["weight"].double() * loss, 0.0)
        return loss.detach(), logp.detach(), torch.where(live, kl, 0.0).detach(), torch.autograd.grad(loss.sum(), x)[0]
    if not c["vocab"]:
        logp = s["logp"].detach().double().requires_grad_(True)
        loss, chosen, rejected = _exact_pairs(c, logp, s["ref"], s["target"], s["offsets"])
        return loss.detach(), chosen, rejected, torch.autograd.grad(loss, logp, s["grad"].double())[0]
    x, logp, _ = _exact_logp(s["logits"], s["target"], 1.0)
    loss, chosen, rejected = _exact_pairs(c, logp, s["ref"], s["target"], s["offsets"])
    return loss.detach(), chosen, rejected, logp.detach(), torch.autograd.grad(loss, x, s["grad"].double())[0]
