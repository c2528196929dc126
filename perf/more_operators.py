"""The dense end of a training step as a training program calls it: losses over a decoder's head without its logits,
and the AdamW step of all dense weights at once. The cases whose time is measured, with their inputs, the work they
cannot do without, their plain form and their results in 64 bits.

Kinds of case (field "kind"):
  logps  head_token_logps: log-probabilities of given tokens from hidden states and head, forward, or with the gradients
         of given token weights
  ce     head_cross_entropy: the mean cross entropy, with label smoothing and a penalty on the log of the softmax's sum
  adamw  DenseAdamW.step: all tensors of a model, moments in 32 bits ("bits" 32) or as 8-bit floats with a
         power-of-two scale for each 128 values (8)

"grads" of the head's cases: "" (forward alone), "hidden" (the head is frozen, as where an engram alone is trained) or
"both". Hidden states are those after a decoder's last norm, N(0, 1) with a part along the target's row of the head that
lets it carry most of the probability; logits are then N(0, 2) beside it. "shift": the hidden states are [:, :-1] of a
longer tensor, as next-token targets make them. Weights, gradients and moments of a model lie in one flat buffer each,
every tensor from a multiple of 128 values on.
"""
import math

import torch

own = False

_DEV = "cuda"
_IGNORE = -100
_LARGE_VOCAB, _LARGE_DIM, _LARGE_MEM = 262_144, 5_376, 1_536  # this repository's large configuration
_SMALL_VOCAB, _SMALL_DIM = 32_000, 1_024                      # its small one


def listed():
    large = dict(vocab=_LARGE_VOCAB, dim=_LARGE_DIM, dtype="bf16")
    small = dict(vocab=_SMALL_VOCAB, dim=_SMALL_DIM, dtype="fp32")
    plain = dict(masked=0.0, temperature=1.0, shift=False)
    ce = dict(plain, kind="ce", smoothing=0.0, z_loss=0.0)
    return [
        # the log-probability of one sampled token of a server of the small model: latency
        dict(small, **plain, name="logps_1", kind="logps", batch=1, seq=1, grads=""),
        # a reference's log-probabilities over a batch of answers, next-token views, prompts left out
        dict(large, name="logps_8x511", kind="logps", batch=8, seq=511, grads="", masked=0.25, temperature=1.0, shift=True),
        # weighted likelihood training of a small fp32 model, odd rows, sampled at a temperature
        dict(small, name="logps_fp32_3x341", kind="logps", batch=3, seq=341, grads="both", masked=0.1, temperature=0.7, shift=False),
        # an engram trained on one short answer under a frozen head
        dict(large, **ce, name="ce_48", batch=1, seq=48, grads="hidden"),
        # the training batch of the large configuration under a frozen head, prompts left out
        dict(large, **dict(ce, masked=0.1), name="ce_8192", batch=4, seq=2048, grads="hidden"),
        # a tied head trained with it, odd rows, smoothed targets and the penalty
        dict(large, **dict(ce, smoothing=0.1, z_loss=1e-4), name="ce_tied_3x683", batch=3, seq=683, grads="both"),
        # the small configuration, everything trained
        dict(small, **ce, name="ce_fp32_2048", batch=1, seq=2048, grads="both"),
        # the dense weights of one engram of the large configuration
        dict(name="adamw_engram", kind="adamw", bits=32, engrams=1, layers=0, dim=_LARGE_DIM, mem=_LARGE_MEM, ffn=0, vocab=0, dtype="bf16", gdtype="bf16", decay=0.0),
        # all weights of a small fp32 decoder
        dict(name="adamw_decoder_fp32", kind="adamw", bits=32, engrams=0, layers=24, dim=_SMALL_DIM, mem=0, ffn=2_816, vocab=_SMALL_VOCAB, dtype="fp32", gdtype="fp32", decay=0.1),
        # four tiny engrams: latency, many small tensors
        dict(name="adamw8_engrams_tiny", kind="adamw", bits=8, engrams=4, layers=0, dim=257, mem=72, ffn=0, vocab=0, dtype="bf16", gdtype="bf16", decay=0.01),
        # a decoder with its engrams, odd widths, 8-bit moments
        dict(name="adamw8_decoder", kind="adamw", bits=8, engrams=2, layers=30, dim=1_531, mem=768, ffn=4_093, vocab=50_021, dtype="bf16", gdtype="bf16", decay=0.1),
        # bf16 weights with gradients summed in fp32, 8-bit moments
        dict(name="adamw8_engrams_2", kind="adamw", bits=8, engrams=2, layers=0, dim=_LARGE_DIM, mem=_LARGE_MEM, ffn=0, vocab=0, dtype="bf16", gdtype="fp32", decay=0.1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same kinds: rows, vocabulary and width over the logarithm of their ranges, odd ones among them;
    models of 1e4 to 9e8 weights."""
    kind = rng.choice(("logps", "ce", "ce", "adamw", "adamw"))
    if kind == "adamw":
        dim = _log_int(rng, 40, 2_048)
        c = dict(kind=kind, bits=rng.choice((8, 8, 32)), engrams=rng.choice((0, 1, 2, 5)), layers=0, dim=dim, mem=8 * _log_int(rng, 4, 192),
                 ffn=0, vocab=0, dtype=rng.choice(("bf16", "bf16", "fp32")), gdtype="bf16", decay=rng.choice((0.0, 0.1)))
        if c["engrams"] == 0 or rng.random() < 0.5:
            layers = rng.choice((1, 4, 13, 32))
            c.update(layers=layers, ffn=rng.choice((4 * dim, dim + 3)), vocab=_log_int(rng, 1_000, 32_000))
        if c["dtype"] == "fp32" or rng.random() < 0.3:
            c["gdtype"] = "fp32"
        while work(c)["bytes"] > 9.2e9:
            c["layers"] //= 2
        return c
    dtype = rng.choice(("bf16", "bf16", "bf16", "fp32"))
    grads = rng.choice(("", "hidden", "hidden", "both"))
    vocab = rng.choice((_LARGE_VOCAB, _SMALL_VOCAB, _log_int(rng, 1_000, 262_144), _log_int(rng, 1_000, 262_144)))
    dim = rng.choice((_LARGE_DIM, _SMALL_DIM, 64 * _log_int(rng, 1, 84), 8 * _log_int(rng, 8, 600), _log_int(rng, 40, 4_000)))
    # at most the largest listed case's products, a third of them in fp32
    most = 16_384 * _LARGE_VOCAB * _LARGE_DIM // (vocab * dim * {"": 1, "hidden": 2, "both": 3}[grads])
    tokens = _log_int(rng, 1, max(1, min(8_192, most if dtype == "bf16" else most // 3)))
    batch = min(tokens, rng.choice((1, 1, 2, 5, 16)))
    c = dict(kind=kind, vocab=vocab, dim=dim, dtype=dtype, grads=grads, batch=batch, seq=tokens // batch, masked=rng.choice((0.0, 0.0, 0.2, 0.5)),
             temperature=rng.choice((1.0, 1.0, 0.7, 2.0)), shift=rng.random() < 0.3)
    if kind == "ce":
        c.update(smoothing=rng.choice((0.0, 0.0, 0.1)), z_loss=rng.choice((0.0, 0.0, 1e-4)))
    return c


# ------------------------------------------------------------------------------------ inputs
def _dtype(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def prepare(case, seed):
    gen = torch.Generator(device=_DEV).manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return torch.empty(shape, device=_DEV).normal_(mean, std, generator=gen)

    return (_prepare_adamw if case["kind"] == "adamw" else _prepare_head)(case, seed, gen, normal)


def _prepare_head(case, seed, gen, normal):
    batch, seq, vocab, dim, dtype = case["batch"], case["seq"], case["vocab"], case["dim"], _dtype(case["dtype"])
    weight = torch.empty((vocab, dim), device=_DEV, dtype=dtype).normal_(0.0, 2.0 / math.sqrt(dim), generator=gen)
    targets = torch.randint(0, vocab, (batch, seq), generator=gen, device=_DEV)
    row = weight[targets.reshape(-1)].float()
    row = row / row.square().sum(1, keepdim=True).sqrt()
    raised = normal(batch * seq, 1, std=0.75, mean=0.5 * (math.log(vocab) + 2.0))
    hidden = (normal(batch * seq, dim) + raised * row).to(dtype).view(batch, seq, dim)
    if case["shift"]:  # one more token of each sequence, which predicts nothing
        hidden = torch.cat([hidden, hidden[:, -1:]], dim=1)[:, :-1]
    targets[:, :int(case["masked"] * seq)] = _IGNORE
    state = {"case": case, "targets": targets, "hidden": hidden.detach(), "weight": weight}
    if case["grads"]:
        state["hidden"].requires_grad_()
    if case["grads"] == "both":
        weight.requires_grad_()
    if case["kind"] == "logps":
        state["upstream"] = torch.rand((batch, seq), generator=gen, device=_DEV)
    return state


_BLOCK = 128
_LR, _BETA1, _BETA2, _EPS, _STEP = 1e-3, 0.9, 0.999, 1e-8, 10


def _shapes(case):
    d, shapes = case["dim"], []
    for _ in range(case["engrams"]):
        shapes += [(d, case["mem"]), (d, case["mem"]), (d,), (d,)]
    for _ in range(case["layers"]):
        shapes += [(d, d)] * 4 + [(case["ffn"], d)] * 2 + [(d, case["ffn"])] + [(d,)] * 2
    if case["vocab"]:
        shapes += [(case["vocab"], d), (d,)]
    return shapes


def _places(case):
    """[(first value in the flat buffers, shape)], length of the flat buffers."""
    at, places = 0, []
    for shape in _shapes(case):
        places.append((at, shape))
        at += -(-math.prod(shape) // _BLOCK) * _BLOCK
    return places, at


def _prepare_adamw(case, seed, gen, normal):
    places, total = _places(case)
    sizes = torch.tensor([math.prod(s) for _, s in places], device=_DEV)
    starts = torch.tensor([a for a, _ in places], device=_DEV)
    # tensor and place in it of each eight values: what the rounding's random numbers are counted by
    groups = torch.arange(total // 8, device=_DEV) * 8
    stream = torch.searchsorted(starts, groups, right=True) - 1
    inside = groups - starts[stream]
    real = ((inside[:, None] + torch.arange(8, device=_DEV)) < sizes[stream][:, None]).view(-1)
    state = {"case": case, "seed": seed * 7_919 + 5, "step": _STEP, "stream": stream, "group": inside // 8}
    state["p"] = torch.where(real, normal(total, std=0.02), 0.0).to(_dtype(case["dtype"]))
    # each value's gradients have a size of its own, log-normal
    size = torch.exp(normal(total, std=1.0) - 7.0)
    state["g"] = torch.where(real, normal(total) * size, 0.0).to(_dtype(case["gdtype"]))
    m, v = torch.where(real, 0.3 * normal(total) * size, 0.0), torch.where(real, size * size * torch.exp(normal(total, std=0.3)), 0.0)
    if case["bits"] == 32:
        state["m"], state["v"] = m, v
    else:
        noise = torch.full((total,), 1 << 15, dtype=torch.int32, device=_DEV)
        (state["m"], state["m_scale"]), (state["v"], state["v_scale"]) = _to8(m, noise, False), _to8(v, noise, True)
    state["places"] = places
    return state


# ------------------------------------------------------------------------------------ one pass
def run(state):
    kind = state["case"]["kind"]
    return (_OWN if own else _PLAIN)[kind](state)


def _own_logps(state):
    from micro_engram_fork_amd import losses

    case = state["case"]
    logps = losses.head_token_logps(state["hidden"], state["weight"], state["targets"], temperature=case["temperature"])
    out = {"logps": logps}
    if case["grads"]:
        wanted = [state[k] for k in _wanted(case)]
        out.update(zip(_wanted(case), torch.autograd.grad(logps, wanted, state["upstream"])))
    return out


def _own_ce(state):
    from micro_engram_fork_amd import losses

    case = state["case"]
    loss = losses.head_cross_entropy(state["hidden"], state["weight"], state["targets"], temperature=case["temperature"],
                                     label_smoothing=case["smoothing"], z_loss=case["z_loss"])
    out = {"loss": loss}
    if case["grads"]:
        out.update(zip(_wanted(case), torch.autograd.grad(loss, [state[k] for k in _wanted(case)])))
    return out


def _wanted(case):
    return {"": (), "hidden": ("hidden",), "both": ("hidden", "weight")}[case["grads"]]


def _optimizer(state):
    """The optimizer of the state's tensors, which a program makes once."""
    from micro_engram_fork_amd import optim

    case, params = state["case"], []
    for at, shape in state["places"]:
        n = math.prod(shape)
        p = torch.nn.Parameter(state["p"][at:at + n].view(shape))
        if case["dtype"] == case["gdtype"]:
            p.grad = state["g"][at:at + n].view(shape)
        else:  # sums of several backwards, in a type that torch lets no bf16 parameter's grad have
            p.fp32_grad = state["g"][at:at + n].view(shape)
        params.append(p)
    opt = optim.DenseAdamW(params, lr=_LR, betas=(_BETA1, _BETA2), eps=_EPS, weight_decay=case["decay"], state_bits=case["bits"], seed=state["seed"])
    for (at, shape), p in zip(state["places"], params):
        n = math.prod(shape)
        opt.state[p].update(step=torch.tensor(float(_STEP)), exp_avg=state["m"][at:at + n].view(shape), exp_avg_sq=state["v"][at:at + n].view(shape))
        if case["bits"] == 8:
            b = slice(at // _BLOCK, -(-(at + n) // _BLOCK))
            opt.state[p].update(exp_avg_scale=state["m_scale"][b], exp_avg_sq_scale=state["v_scale"][b])
    return opt


def _own_adamw(state):
    if "optimizer" not in state:
        state["optimizer"] = _optimizer(state)
    state["optimizer"].step()
    return _adamw_outputs(state)


def _adamw_outputs(state):
    return {k: state[k] for k in ("p", "m", "v", "m_scale", "v_scale") if k in state}


# --- plain: the head
def _logits(state):
    """(hidden states of the rows [n, dim], logits / temperature [n, vocab], both fp32, targets, rows that count)."""
    case = state["case"]
    h = state["hidden"].detach().reshape(-1, case["dim"]).float()
    t = state["targets"].reshape(-1, 1)
    valid = (t >= 0) & (t < case["vocab"])
    h = torch.where(valid, h, 0.0)
    z = (h @ state["weight"].detach().float().t()) * (1.0 / case["temperature"])
    return h, z, t.clamp(0, case["vocab"] - 1), valid.squeeze(1)


def _softmax(z):
    """(exponentials' share of their sum, log of the sum)."""
    top = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - top)
    s = e.sum(dim=1, keepdim=True)
    return e / s, (torch.log(s) + top).squeeze(1)


def _head_grads(state, out, g, h):
    """g: the gradient of the logits before the temperature, fp32."""
    case = state["case"]
    out["hidden"] = (g @ state["weight"].detach().float()).to(state["hidden"].dtype).view(state["hidden"].shape)
    if case["grads"] == "both":
        out["weight"] = (g.t() @ h).to(state["weight"].dtype)
    return out


def _plain_logps(state):
    case = state["case"]
    h, z, t, valid = _logits(state)
    q, lse = _softmax(z)
    out = {"logps": torch.where(valid, z.gather(1, t).squeeze(1) - lse, 0.0).view(state["targets"].shape)}
    if not case["grads"]:
        return out
    coef = torch.where(valid, state["upstream"].reshape(-1), 0.0)[:, None] * (1.0 / case["temperature"])
    return _head_grads(state, out, (-coef * q).scatter_add_(1, t, coef), h)


def _plain_ce(state):
    case = state["case"]
    eps, penalty = case["smoothing"], case["z_loss"]
    h, z, t, valid = _logits(state)
    q, lse = _softmax(z)
    each = lse - (1 - eps) * z.gather(1, t).squeeze(1) + penalty * lse * lse
    if eps:
        each = each - eps / case["vocab"] * z.sum(dim=1)
    count = valid.float().sum().clamp(min=1.0)
    out = {"loss": torch.where(valid, each, 0.0).sum() / count}
    if not case["grads"]:
        return out
    g = q * (1 + 2 * penalty * lse)[:, None]
    if eps:
        g = g - eps / case["vocab"]
    g.scatter_add_(1, t, torch.full_like(t, -(1 - eps), dtype=torch.float32))
    return _head_grads(state, out, g * (valid.float() / (count * case["temperature"]))[:, None], h)


# --- plain: AdamW
def _noise(state):
    """16 random bits for each value: Philox4x32-10 (Salmon et al. 2011) of (its place in its tensor / 8, step, tensor),
    keyed by the seed."""
    mask = 0xffffffff
    zero = torch.zeros_like(state["group"])
    c = [state["group"] & mask, state["group"] >> 32, zero + state["step"], state["stream"]]
    k0, k1 = state["seed"] & mask, state["seed"] >> 32
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & mask) ^ c[1] ^ k0, b & mask, ((a >> 32) & mask) ^ c[3] ^ k1, a & mask]
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    halves = torch.stack([x for w in c for x in (w & 0xffff, w >> 16)], dim=1)
    return halves.view(-1).int()


def _to8(x, noise, second):
    """(8-bit floats, scale of each block): stochastic rounding of x / scale, the scale a power of two that puts the
    block's largest value in the binade of 2^7 (e4m3) or, for second moments (e5m2), 2^14. A second moment over zero
    stays over zero."""
    bits, lowest, top = (2, -14, 14) if second else (3, -6, 7)
    blocks = x.view(-1, _BLOCK)
    exponent = blocks.abs().amax(dim=1).view(torch.int32) >> 23
    scale = (exponent - top).clamp(min=0)
    y = torch.ldexp(blocks.abs(), (127 - scale)[:, None]).view(-1)
    drop = 23 - bits
    add = (noise << (drop - 16)) + (1 << (drop - 17))
    code = ((y.view(torch.int32) + add) >> drop) - ((126 + lowest) << bits)
    small = (y * 2.0 ** (bits - lowest) + add.float() * 2.0 ** -drop).int()
    code = torch.where(y < 2.0 ** lowest, small, code)
    if second:
        code = torch.where((code == 0) & (x > 0), 1, code)
    else:
        code = torch.where(x < 0, code + 128, code)
    kind = torch.float8_e5m2 if second else torch.float8_e4m3fn
    return code.to(torch.uint8).view(kind), scale.to(torch.uint8).view(torch.float8_e8m0fnu)


def _from8(x, scale):
    two = torch.full_like(scale, 1.0, dtype=torch.float32)
    return (x.float().view(-1, _BLOCK) * torch.ldexp(two, scale.view(torch.uint8).int() - 127)[:, None]).view(-1)


def _plain_adamw(state):
    case = state["case"]
    state["step"] += 1
    t = state["step"]
    p, g = state["p"].float(), state["g"].float()
    m, v = (state["m"], state["v"]) if case["bits"] == 32 else (_from8(state["m"], state["m_scale"]), _from8(state["v"], state["v_scale"]))
    noise = _noise(state) if case["bits"] == 8 or case["dtype"] == "bf16" else None
    m = _BETA1 * m + (1 - _BETA1) * g
    v = _BETA2 * v + (1 - _BETA2) * (g * g)
    size = _LR / (1 - _BETA1 ** t)
    p = p * (1 - _LR * case["decay"]) - size * (m / (torch.sqrt(v) / math.sqrt(1 - _BETA2 ** t) + _EPS))
    if case["dtype"] == "bf16":
        p = ((p.view(torch.int32) + noise) & -65536).view(torch.float32)
    state["p"].copy_(p)
    if case["bits"] == 32:
        state["m"].copy_(m), state["v"].copy_(v)
    else:
        turned = ((noise << 8) | (noise >> 8)) & 0xffff
        for name, new in zip(("m", "v"), (_to8(m, turned, False), _to8(v, 0xffff - noise, True))):
            state[name].view(torch.uint8).copy_(new[0].view(torch.uint8))
            state[name + "_scale"].view(torch.uint8).copy_(new[1].view(torch.uint8))
    return _adamw_outputs(state)


_OWN = {"logps": _own_logps, "ce": _own_ce, "adamw": _own_adamw}
_PLAIN = {"logps": _plain_logps, "ce": _plain_ce, "adamw": _plain_adamw}


# ------------------------------------------------------------------------------------ work
def work(case):
    """Head: hidden states of the rows that count and head read once, gradients written once, one product of rows and
    head for the logits and one for each gradient. AdamW: weights and moments read and written, gradients read."""
    if case["kind"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        p, g = (2 if case[k] == "bf16" else 4 for k in ("dtype", "gdtype"))
        moments = 2 * 4 if case["bits"] == 32 else 2 * (1 + 1 / _BLOCK)
        return {"bytes": n * (2 * p + g + 2 * moments), "flops": 15 * n}
    size, vocab, dim, rows = (2 if case["dtype"] == "bf16" else 4), case["vocab"], case["dim"], case["batch"] * case["seq"]
    counted = case["batch"] * (case["seq"] - int(case["masked"] * case["seq"]))
    made = {"": 0, "hidden": rows * dim, "both": (rows + vocab) * dim}[case["grads"]]
    return {"bytes": size * ((counted + vocab) * dim + made) + 12 * rows,
            "flops": 2 * counted * vocab * dim * (1 + len(_wanted(case))) + 4 * counted * vocab}


# ------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return _exact_adamw(case, state) if case["kind"] == "adamw" else _exact_head(case, state)


def _exact_head(case, state):
    """The definitions in float64, a block of rows at a time."""
    vocab, dim, temp = case["vocab"], case["dim"], case["temperature"]
    hidden, targets = state["hidden"].detach().reshape(-1, dim), state["targets"].reshape(-1)
    weight = state["weight"].detach().double()
    n, where = hidden.shape[0], (targets != _IGNORE).nonzero().squeeze(1)
    each = torch.zeros(n, dtype=torch.float64, device=_DEV)
    grad_h = torch.zeros((n, dim), dtype=torch.float64, device=_DEV) if case["grads"] else None
    grad_w = torch.zeros((vocab, dim), dtype=torch.float64, device=_DEV) if case["grads"] == "both" else None
    eps, penalty = case.get("smoothing", 0.0), case.get("z_loss", 0.0)
    for rows in where.split(max(1, (1 << 28) // vocab)):
        h = hidden[rows].double()
        logits = (h @ weight.t()).div_(temp)
        lse = torch.logsumexp(logits, dim=1)
        at = (torch.arange(rows.numel(), device=_DEV), targets[rows])
        picked = logits[at]
        if case["kind"] == "logps":
            each[rows] = picked - lse
            scale = -state["upstream"].reshape(-1)[rows].double()
        else:
            each[rows] = lse - (1 - eps) * picked - eps * logits.mean(dim=1) + penalty * lse.square()
            scale = torch.full_like(lse, 1.0 / where.numel())
        if grad_h is None:
            continue
        d = logits.sub_(lse[:, None]).exp_().mul_((1 + 2 * penalty * lse)[:, None]).sub_(eps / vocab)
        d[at] -= 1 - eps
        d.mul_((scale / temp)[:, None])
        grad_h[rows] = d @ weight
        if grad_w is not None:
            grad_w += d.t() @ h
    out = {"logps": each.view(state["targets"].shape)} if case["kind"] == "logps" else {"loss": each.sum() / max(1, where.numel())}
    if grad_h is not None:
        out["hidden"] = grad_h.view(state["hidden"].shape)
    if grad_w is not None:
        out["weight"] = grad_w
    return out


def _exact_adamw(case, state):
    """Weights (and 32-bit moments) before any rounding; what a rounded moment should be has no value of its own."""
    t, g = _STEP + 1, state["g"].double()

    def moment(name):
        if case["bits"] == 32:
            return state[name].double()
        scale = torch.exp2(state[name + "_scale"].view(torch.uint8).double() - 127).repeat_interleave(_BLOCK)
        return state[name].double() * scale

    m = torch.lerp(g, moment("m"), _BETA1)
    v = torch.lerp(g.square(), moment("v"), _BETA2)
    update = (m / (1 - _BETA1 ** t)) / ((v / (1 - _BETA2 ** t)).sqrt() + _EPS)
    p = state["p"].double()
    out = {"p": p - _LR * case["decay"] * p - _LR * update, "m": None, "v": None}
    if case["bits"] == 32:
        out.update(m=m, v=v)
    else:
        out.update(m_scale=None, v_scale=None)
    return out
