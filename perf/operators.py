"""The losses over a decoder's logits as a training program calls them: the cases whose time is measured, with their
inputs, the work they cannot do without, their plain form and their results in 64 bits.

Kinds of case (field "kind"):
  logps       token_logps: log-probabilities of given tokens, forward, or with the gradient of given token weights
  distill     distill_loss: from a teacher's top logits, renormalised or with the rest as one class ("rest")
  preference  preference_loss: packed sequences, the first half chosen, the second half rejected
  policy      policy_loss: clipped ratios and a KL term on sampled answers

"train" cases return the loss and the gradient of the logits, the others the loss alone. Logits are those of a
decoder: N(0, 2) over the vocabulary with a few tokens raised to carry most of the probability. "pad": columns of a padded
vocabulary that the logits are a view without; "shift": the logits are [:, :-1] of a longer tensor, as next-token targets make them.
"""
import math
import random

import torch

own = False

_DEV = "cuda"
_IGNORE = -100
_LARGE_VOCAB = 262_144  # this repository's large configuration
_SMALL_VOCAB = 32_000   # its small one


def listed():
    return [
        # the log-probability of one sampled token of a server: latency
        dict(name="logps_1", kind="logps", batch=1, seq=1, vocab=_LARGE_VOCAB, dtype="bf16", train=False, pad=0, shift=False, masked=0.0, temperature=1.0),
        # a reference's log-probabilities over a batch of answers, next-token views of the logits, prompts left out
        dict(name="logps_8x511", kind="logps", batch=8, seq=511, vocab=_LARGE_VOCAB, dtype="bf16", train=False, pad=0, shift=True, masked=0.25, temperature=1.0),
        # weighted likelihood training of a small fp32 model
        dict(name="logps_fp32_3x341", kind="logps", batch=3, seq=341, vocab=_SMALL_VOCAB, dtype="fp32", train=True, pad=0, shift=False, masked=0.1, temperature=1.0),
        # distillation on one short answer
        dict(name="distill_48", kind="distill", batch=1, seq=48, vocab=_LARGE_VOCAB, dtype="bf16", train=True, top=20, rest=False, pad=0, masked=0.0, temperature=1.0),
        # distillation over a packed sequence, the rest of the vocabulary as one class
        dict(name="distill_4096", kind="distill", batch=1, seq=4096, vocab=_LARGE_VOCAB, dtype="bf16", train=True, top=64, rest=True, pad=0, masked=0.2, temperature=2.0),
        # fp32, odd vocabulary: rows that start at any 4-byte address
        dict(name="distill_fp32_2x1531", kind="distill", batch=2, seq=1531, vocab=32_003, dtype="fp32", train=True, top=8, rest=False, pad=0, masked=0.0, temperature=1.5),
        # two pairs of short answers
        dict(name="preference_2", kind="preference", pairs=2, longest=40, vocab=_SMALL_VOCAB, dtype="bf16", train=True, loss="sigmoid", smoothing=0.0, normalized=False, pad=0),
        # a whole preference batch, ragged answers
        dict(name="preference_12", kind="preference", pairs=12, longest=512, vocab=_LARGE_VOCAB, dtype="bf16", train=True, loss="sigmoid", smoothing=0.1, normalized=False, pad=0),
        # evaluation on held-out pairs, odd vocabulary, logits cut from a padded head
        dict(name="preference_eval_5", kind="preference", pairs=5, longest=300, vocab=131_075, dtype="bf16", train=False, loss="ipo", smoothing=0.0, normalized=True, pad=61),
        # a few sampled tokens of one answer
        dict(name="policy_16", kind="policy", batch=1, seq=16, vocab=_LARGE_VOCAB, dtype="bf16", train=True, reference=True, reduction="token", pad=0, masked=0.0, temperature=1.0),
        # a group of long answers, with a reference
        dict(name="policy_16x512", kind="policy", batch=16, seq=512, vocab=_LARGE_VOCAB, dtype="bf16", train=True, reference=True, reduction="token", pad=0, masked=0.2, temperature=1.0),
        # fp32, odd sizes, every answer weighted alike, sampled at a temperature
        dict(name="policy_fp32_5x777", kind="policy", batch=5, seq=777, vocab=50_021, dtype="fp32", train=True, reference=False, reduction="sequence", pad=0, masked=0.15, temperature=0.7),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same kinds: rows and vocabulary over the logarithm of their ranges, odd ones among them, at most
    1.2e9 logits (fp32: 6e8)."""
    kind = rng.choice(("logps", "distill", "preference", "policy"))
    dtype = rng.choice(("bf16", "bf16", "bf16", "fp32"))
    vocab = rng.choice((_LARGE_VOCAB, _SMALL_VOCAB, _log_int(rng, 1_000, 262_144), _log_int(rng, 1_000, 262_144)))
    most = max(4, min(8_192, (1_200_000_000 if dtype == "bf16" else 600_000_000) // vocab))
    c = dict(kind=kind, vocab=vocab, dtype=dtype, train=rng.random() < 0.75, pad=rng.choice((0, 0, 0, 13, 128)))
    if kind == "preference":
        c["pairs"] = rng.choice((1, 2, 3, 8, 13))
        c["longest"] = _log_int(rng, 2, max(2, min(2_048, most // (2 * c["pairs"]))))
        return dict(c, loss=rng.choice(("sigmoid", "sigmoid", "ipo", "hinge")), smoothing=0.0, normalized=rng.random() < 0.4)
    tokens = _log_int(rng, 1, most)
    c["batch"] = min(tokens, rng.choice((1, 1, 2, 5, 16)))
    c["seq"] = tokens // c["batch"]
    c["masked"] = rng.choice((0.0, 0.0, 0.2, 0.5))
    c["temperature"] = rng.choice((1.0, 1.0, 0.7, 2.0))
    if kind == "logps":
        return dict(c, shift=rng.random() < 0.3)
    if kind == "distill":
        return dict(c, top=rng.choice((1, 5, 8, 20, 64, 100)), rest=rng.random() < 0.5)
    return dict(c, reference=rng.random() < 0.6, reduction=rng.choice(("token", "sequence")))


# ------------------------------------------------------------------------------------ inputs
def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _lengths(case):
    """Lengths of a preference batch's sequences and of their prompts: part of the case, not of its seed."""
    r = random.Random(case["pairs"] * 1_000_003 + case["longest"])
    lengths = [r.randint(max(1, case["longest"] // 3), case["longest"]) for _ in range(2 * case["pairs"])]
    return lengths, [n // 5 for n in lengths]


def _rows(case):
    return sum(_lengths(case)[0]) if case["kind"] == "preference" else case["batch"] * case["seq"]


def _counted(case):
    """Rows that count in the loss: the first tokens of each sequence are its prompt and do not."""
    if case["kind"] == "preference":
        lengths, prompts = _lengths(case)
        return sum(lengths) - sum(prompts)
    return case["batch"] * (case["seq"] - int(case["masked"] * case["seq"]))


def _logits(case, gen, raised, heights):
    """Logits in the shape and memory layout of the case: N(0, 2), and `raised` [rows, r] at `heights` above the
    level at which one token holds as much as all others together."""
    vocab, rows = case["vocab"], _rows(case)
    x = torch.empty((rows, vocab), device=_DEV, dtype=torch.float32).normal_(0.0, 2.0, generator=gen)
    x.scatter_(1, raised, heights + (math.log(vocab) + 2.0))
    x = x.to(_dtype(case))
    if case["kind"] != "preference":
        x = x.view(case["batch"], case["seq"], vocab)
    if case.get("shift"):  # one more token of each sequence, whose logits predict nothing
        x = torch.cat([x, x[:, -1:]], dim=1)[:, :-1]
    if case["pad"]:
        wide = x.new_empty((*x.shape[:-1], vocab + case["pad"]))
        wide[..., :vocab] = x
        x = wide[..., :vocab]
    return x.requires_grad_() if case["train"] else x


def prepare(case, seed):
    gen = torch.Generator(device=_DEV).manual_seed(seed)
    vocab, rows, kind = case["vocab"], _rows(case), case["kind"]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.empty(shape, device=_DEV).normal_(mean, std, generator=gen)

    state = {"case": case}
    if kind == "distill":
        k = min(case["top"], vocab // 2)
        start = torch.randint(0, vocab, (rows, 1), generator=gen, device=_DEV)
        ids = (start + torch.randint(1, vocab // k + 1, (rows, k), generator=gen, device=_DEV).cumsum(1)) % vocab
        rank = torch.arange(1, k + 1, device=_DEV, dtype=torch.float32)
        teacher, _ = (normal(rows, k, std=0.7) - 1.5 * rank.log() + 20.0).sort(dim=1, descending=True)
        state["logits"] = _logits(case, gen, ids, 0.8 * (teacher - 20.0) + normal(rows, k, std=0.5))
        shape = (case["batch"], case["seq"])
        state["ids"] = ids.view(*shape, k)
        state["teacher"] = teacher.to(_dtype(case)).view(*shape, k)
        state["teacher_lse"] = None
        if case["rest"]:  # the teacher's own tokens outside its top ones hold about a tenth
            top = (state["teacher"].float() / case["temperature"]).logsumexp(-1)
            state["teacher_lse"] = top + 0.05 + 0.1 * torch.rand(shape, generator=gen, device=_DEV)
        state["mask"] = None
        if case["masked"]:
            state["mask"] = (torch.arange(case["seq"], device=_DEV) >= int(case["masked"] * case["seq"])).expand(shape).contiguous()
        return state
    targets = torch.randint(0, vocab, (rows, 1), generator=gen, device=_DEV)
    state["logits"] = _logits(case, gen, targets, normal(rows, 1, std=1.5, mean=0.5))
    if kind == "preference":
        lengths, prompts = _lengths(case)
        targets = targets.view(rows)
        starts = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
        inside = torch.zeros(rows, dtype=torch.bool)
        for a, p in zip(starts, prompts):
            inside[a:a + p] = True
        state["targets"] = targets.masked_fill(inside.to(_DEV), _IGNORE)
        state["cu_seqlens"] = torch.tensor(starts, dtype=torch.int32, device=_DEV)
        near = 0.1
    else:
        shape = (case["batch"], case["seq"])
        state["targets"] = targets.view(shape).clone()
        state["targets"][:, :int(case["masked"] * case["seq"])] = _IGNORE
        near = 0.1 / case["temperature"]
    # what an earlier form of the model gave these tokens: near, not equal
    flat = state["logits"].detach().reshape(rows, vocab).float() / case.get("temperature", 1.0)
    now = (flat.gather(1, targets.view(rows, 1)).squeeze(1) - flat.logsumexp(1)).view(state["targets"].shape)
    del flat
    if kind == "logps":
        state["weights"] = torch.rand(now.shape, generator=gen, device=_DEV)
    elif kind == "preference":
        # training has moved the chosen answers up and the rejected ones down
        moved = torch.where(torch.arange(rows, device=_DEV) < starts[case["pairs"]], 0.03, -0.03)
        state["ref_logps"] = now - moved + normal(rows, std=near)
    else:
        state["old_logps"] = now + normal(*now.shape, std=near)
        state["ref_logps"] = now + normal(*now.shape, std=2 * near) if case["reference"] else None
        state["advantages"] = normal(case["batch"])  # one for each answer
    return state


# ------------------------------------------------------------------------------------ one pass
_LO, _HI, _KL, _BETA = 0.2, 0.28, 0.04, 0.1


def run(state):
    kind = state["case"]["kind"]
    return _run_own(state, kind) if own else _PLAIN[kind](state)


def _run_own(state, kind):
    from micro_engram_fork_amd import losses

    case, logits = state["case"], state["logits"]
    if kind == "logps":
        logps = losses.token_logps(logits, state["targets"], temperature=case["temperature"])
        if not case["train"]:
            return {"logps": logps}
        grad, = torch.autograd.grad(logps, logits, state["weights"])
        return {"logps": logps, "grad": grad}
    if kind == "distill":
        loss = losses.distill_loss(logits, state["ids"], state["teacher"], teacher_lse=state["teacher_lse"], mask=state["mask"],
                                   temperature=case["temperature"])
        out = {"loss": loss}
    elif kind == "preference":
        loss, chosen, rejected = losses.preference_loss(logits, state["targets"], state["ref_logps"], cu_seqlens=state["cu_seqlens"],
                                                        beta=_BETA, loss_type=case["loss"], label_smoothing=case["smoothing"],
                                                        length_normalized=case["normalized"])
        out = {"loss": loss, "chosen": chosen, "rejected": rejected}
    else:
        loss, logps, stats = losses.policy_loss(logits, state["targets"], state["old_logps"], state["advantages"],
                                                ref_logps=state["ref_logps"], clip_low=_LO, clip_high=_HI,
                                                kl_coef=_KL if case["reference"] else 0.0, temperature=case["temperature"],
                                                reduction=case["reduction"])
        out = {"loss": loss, "logps": logps, "stats": stats}
    if case["train"]:
        out["grad"], = torch.autograd.grad(loss, logits)
    return out


def _softmax_parts(logits, temperature):
    """(z - max, its exponentials, their sum) in fp32, flat [rows, vocab]."""
    z = logits.detach().reshape(-1, logits.shape[-1]).float()
    z = z * (1.0 / temperature)
    z = z - z.amax(dim=1, keepdim=True)
    e = torch.exp(z)
    return z, e, e.sum(dim=1, keepdim=True)


def _token_parts(logits, targets, temperature):
    """(log-probabilities of the targets, probabilities, targets clamped, rows that count)."""
    z, e, s = _softmax_parts(logits, temperature)
    t = targets.reshape(-1, 1)
    valid = (t >= 0) & (t < logits.shape[-1])
    t = t.clamp(0, logits.shape[-1] - 1)
    logps = torch.where(valid, z.gather(1, t) - torch.log(s), 0.0)
    return logps.squeeze(1), e / s, t, valid.squeeze(1)


def _token_grad(logits, probs, t, coef):
    """coef (1[j = t] - q_j) in the logits' type and shape."""
    g = -coef[:, None] * probs
    g.scatter_add_(1, t, coef[:, None])
    return g.to(logits.dtype).view(logits.shape)


def _plain_logps(state):
    case, logits = state["case"], state["logits"]
    logps, probs, t, valid = _token_parts(logits, state["targets"], case["temperature"])
    out = {"logps": logps.view(state["targets"].shape)}
    if case["train"]:
        coef = torch.where(valid, state["weights"].reshape(-1), 0.0) / case["temperature"]
        out["grad"] = _token_grad(logits, probs, t, coef)
    return out


def _plain_distill(state):
    case, logits = state["case"], state["logits"]
    temp, k = case["temperature"], state["ids"].shape[-1]
    z, e, s = _softmax_parts(logits, temp)
    ids = state["ids"].reshape(-1, k)
    t = state["teacher"].reshape(-1, k).float() * (1.0 / temp)
    valid = torch.ones_like(ids[:, 0], dtype=torch.bool) if state["mask"] is None else state["mask"].reshape(-1)
    if state["teacher_lse"] is None:
        top = t.amax(dim=1, keepdim=True)
        p = torch.exp(t - top)
        p = p / p.sum(dim=1, keepdim=True)
    else:
        p = torch.exp(t - state["teacher_lse"].reshape(-1, 1))
    logq = z.gather(1, ids) - torch.log(s)
    losses = (p * (torch.log(p) - logq)).sum(dim=1)
    weight = valid.float() / valid.float().sum().clamp(min=1.0)
    share = torch.ones_like(s)
    if state["teacher_lse"] is not None:
        r = (1.0 - p.sum(dim=1, keepdim=True)).clamp(min=0.0)
        rest = e.scatter(1, ids, 0.0).sum(dim=1, keepdim=True) / s
        losses = losses + (r * (torch.log(r) - torch.log(rest))).squeeze(1)
        share = (rest - r) / rest
    out = {"loss": (losses * weight).sum() * temp ** 2}
    if case["train"]:
        probs = e / s
        at = probs.gather(1, ids) - p
        grad = (share * probs).scatter(1, ids, at) * (weight * temp)[:, None]
        out["grad"] = grad.to(logits.dtype).view(logits.shape)
    return out


def _plain_preference(state):
    case, logits = state["case"], state["logits"]
    logps, probs, t, valid = _token_parts(logits, state["targets"], 1.0)
    pairs, cu = case["pairs"], state["cu_seqlens"].long()
    rows = torch.arange(logps.shape[0], device=logps.device)
    seq = (rows[:, None] >= cu[None, 1:]).sum(dim=1)
    gap = torch.where(valid, logps - state["ref_logps"], 0.0)
    sums = torch.zeros(2 * pairs, device=logps.device).index_add(0, seq, gap)
    lengths = torch.zeros(2 * pairs, device=logps.device).index_add(0, seq, valid.float()).clamp(min=1.0)
    if case["normalized"]:
        sums = sums / lengths
    h = sums[:pairs] - sums[pairs:]
    x, eps = _BETA * h, case["smoothing"]
    if case["loss"] == "sigmoid":  # log(1 + exp(-x)) without overflow
        soft = torch.log1p(torch.exp(-x.abs()))
        each = (1 - eps) * (soft + (-x).clamp(min=0.0)) + eps * (soft + x.clamp(min=0.0))
        slope = _BETA * (1.0 / (1.0 + torch.exp(-x)) - (1 - eps))
    elif case["loss"] == "ipo":
        each = (h - 0.5 / _BETA) ** 2
        slope = 2 * (h - 0.5 / _BETA)
    else:
        each = (1 - x).clamp(min=0.0)
        slope = torch.where(x < 1, -_BETA, 0.0)
    out = {"loss": each.sum() / pairs, "chosen": _BETA * sums[:pairs], "rejected": _BETA * sums[pairs:]}
    if case["train"]:
        slope = torch.cat([slope, -slope]) / pairs
        if case["normalized"]:
            slope = slope / lengths
        out["grad"] = _token_grad(logits, probs, t, torch.where(valid, slope[seq], 0.0))
    return out


def _plain_policy(state):
    case, logits = state["case"], state["logits"]
    logps, probs, t, valid = _token_parts(logits, state["targets"], case["temperature"])
    shape = state["targets"].shape
    logps, valid = logps.view(shape), valid.view(shape)
    adv = state["advantages"][:, None]
    ratio = torch.exp(logps - state["old_logps"])
    held = ratio.clamp(1 - _LO, 1 + _HI)
    free = ratio * adv <= held * adv
    each = -torch.where(free, ratio * adv, held * adv)
    slope = torch.where(free, -ratio * adv, 0.0)
    kl = torch.zeros_like(each)
    if case["reference"]:
        d = state["ref_logps"] - logps
        kl = torch.expm1(d) - d
        each = each + _KL * kl
        slope = slope - _KL * torch.expm1(d)
    n = valid.float().sum(dim=1, keepdim=True)
    if case["reduction"] == "token":
        weight = valid.float() / n.sum().clamp(min=1.0)
    else:
        weight = valid.float() / n.clamp(min=1.0) / (n > 0).float().sum().clamp(min=1.0)
    count = valid.float().sum().clamp(min=1.0)
    stats = torch.stack([torch.where(valid, kl, 0.0).sum() / count, (valid & ~free).float().sum() / count])
    out = {"loss": torch.where(valid, each * weight, 0.0).sum(), "logps": torch.where(valid, logps, 0.0), "stats": stats}
    if case["train"]:
        coef = torch.where(valid, slope * weight, 0.0).reshape(-1) / case["temperature"]
        out["grad"] = _token_grad(logits, probs, t, coef)
    return out


_PLAIN = {"logps": _plain_logps, "distill": _plain_distill, "preference": _plain_preference, "policy": _plain_policy}


# ------------------------------------------------------------------------------------ work
def work(case):
    """Logits of the rows that count read once, the gradient of every row written once; the tokens' own values are
    small beside them. Operations: scale, difference, exponential and sum for each logit, and three more for its gradient."""
    size, vocab, rows, counted = (2 if case["dtype"] == "bf16" else 4), case["vocab"], _rows(case), _counted(case)
    values = {"logps": 12, "preference": 12, "policy": 20, "distill": 4 + case.get("top", 0) * (8 + size)}[case["kind"]]
    grad = size * vocab * rows if case["train"] else 0
    return {"bytes": size * vocab * counted + grad + values * rows, "flops": vocab * counted * (7 if case["train"] else 4)}


# ------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """The definitions in float64, a block of rows at a time, from log_softmax and autograd of the short formulas on the
    log-probabilities alone."""
    state = prepare(case, seed)
    logits = state["logits"].detach().reshape(-1, case["vocab"])
    shape, temp, n = state["logits"].shape, case.get("temperature", 1.0), logits.shape[0]
    block = max(1, (1 << 28) // case["vocab"])
    spans = [(a, min(n, a + block)) for a in range(0, n, block)]

    def log_softmax(a, b):
        return torch.log_softmax(logits[a:b].double() / temp, dim=1)

    if case["kind"] == "distill":
        weights = _exact_distill_weights(case, state, n)
        total, grads = torch.zeros((), dtype=torch.float64, device=_DEV), None
        if case["train"]:
            grads = torch.empty((n, case["vocab"]), dtype=torch.float64, device=_DEV)
        for a, b in spans:
            each, grad = _exact_distill(case, state, log_softmax(a, b), a, b)
            total = total + (each * weights[a:b]).sum()
            if grads is not None:
                grads[a:b] = grad * weights[a:b, None]
        out = {"loss": total}
        if grads is not None:
            out["grad"] = grads.view(shape)
        return out
    targets = state["targets"].reshape(-1)
    valid = targets != _IGNORE
    logps = torch.cat([log_softmax(a, b)[torch.arange(b - a, device=_DEV), targets[a:b].clamp(min=0)] for a, b in spans])
    logps = logps.masked_fill(~valid, 0.0).requires_grad_()
    if case["kind"] == "logps":
        out, loss = {"logps": logps.view(state["targets"].shape)}, (logps * state["weights"].reshape(-1).double()).sum()
    elif case["kind"] == "preference":
        out, loss = _exact_preference(case, state, logps, valid)
    else:
        out, loss = _exact_policy(case, state, logps, valid)
    if case["train"]:
        coef, = torch.autograd.grad(loss, logps)
        coef = coef.masked_fill(~valid, 0.0) / temp
        grad = torch.empty((n, case["vocab"]), dtype=torch.float64, device=_DEV)
        for a, b in spans:
            grad[a:b] = -coef[a:b, None] * log_softmax(a, b).exp()
            grad[torch.arange(a, b, device=_DEV), targets[a:b].clamp(min=0)] += coef[a:b]
        out["grad"] = grad.view(shape)
    return {k: v.detach() for k, v in out.items()}


def _exact_distill_weights(case, state, n):
    if state["mask"] is None:
        return torch.full((n,), 1.0 / n, dtype=torch.float64, device=_DEV)
    counts = state["mask"].reshape(-1).double()
    return counts / counts.sum().clamp(min=1)


def _exact_distill(case, state, logq, a, b):
    """(losses, gradients before the rows' weights) of rows a to b, from their log-probabilities."""
    temp, k = case["temperature"], state["ids"].shape[-1]
    ids, teacher = state["ids"].reshape(-1, k)[a:b], state["teacher"].reshape(-1, k)[a:b].double() / temp
    if state["teacher_lse"] is None:
        logp = teacher - teacher.logsumexp(1, keepdim=True)
    else:
        logp = teacher - state["teacher_lse"].reshape(-1, 1)[a:b].double()
    at, q = logq.gather(1, ids), logq.exp()
    each = (logp.exp() * (logp - at)).sum(1)
    if state["teacher_lse"] is not None:
        left, other = 1.0 - logp.exp().sum(1), q.scatter(1, ids, 0.0).sum(1)
        each = each + left * (left.log() - other.log())
        q = q * (1.0 - left / other)[:, None]
    return each * temp ** 2, q.scatter(1, ids, at.exp() - logp.exp()) * temp


def _exact_preference(case, state, logps, valid):
    lengths, _ = _lengths(case)
    per = torch.where(valid, logps - state["ref_logps"].double(), 0.0).split(lengths)
    counts = torch.stack([v.sum() for v in valid.split(lengths)]).clamp(min=1)
    d = torch.stack([x.sum() for x in per])
    if case["normalized"]:
        d = d / counts
    h = d[:case["pairs"]] - d[case["pairs"]:]
    log_sigmoid = torch.nn.functional.logsigmoid
    if case["loss"] == "sigmoid":
        each = -(1 - case["smoothing"]) * log_sigmoid(_BETA * h) - case["smoothing"] * log_sigmoid(-_BETA * h)
    elif case["loss"] == "ipo":
        each = (h - 1 / (2 * _BETA)).square()
    else:
        each = torch.relu(1 - _BETA * h)
    loss = each.mean()
    return {"loss": loss, "chosen": _BETA * d[:case["pairs"]], "rejected": _BETA * d[case["pairs"]:]}, loss


def _exact_policy(case, state, logps, valid):
    shape = state["targets"].shape
    lp, ok = logps.view(shape), valid.view(shape).double()
    adv = state["advantages"].double()[:, None]
    ratio = (lp - state["old_logps"].double()).exp()
    held = torch.minimum(torch.maximum(ratio, torch.full_like(ratio, 1 - _LO)), torch.full_like(ratio, 1 + _HI))
    each = torch.maximum(-ratio * adv, -held * adv)
    kl = torch.zeros_like(each)
    if case["reference"]:
        d = state["ref_logps"].double() - lp
        kl = d.exp() - d - 1
        each = each + _KL * kl
    if case["reduction"] == "token":
        loss = (each * ok).sum() / ok.sum().clamp(min=1)
    else:
        n = ok.sum(1)
        loss = ((each * ok).sum(1) / n.clamp(min=1)).sum() / (n > 0).sum().clamp(min=1)
    clipped = (ratio * adv > held * adv).double()
    stats = torch.stack([(kl * ok).sum(), (clipped * ok).sum()]) / ok.sum().clamp(min=1)
    return {"loss": loss, "logps": lp, "stats": stats}, loss
