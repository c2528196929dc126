"""The losses over logits in float64 on the CPU, from their definitions with torch autograd: what the
HIP kernels' outputs are compared with.

Tolerances (relative to the float64 result), set from the kernels' arithmetic before their first run:
a probability q = exp((x - m) / T) / s in fp32 is off by the rounding of its exponent (two roundings of
|z| <= 2^-24 |z| each; logits here reach |z| = 40 at places that matter: 5e-6), by the exponential's unit
in the last place and by the sums' roundings (fewer than 100 additions in a row, halved by their trees:
below 6e-6): 1.5e-5 in all. A log-probability has the same absolute error (d log s = ds / s) and the roundings of
itself. A gradient c (1[j=t] - q) has it relative to |c| times (q, or 1 at the target), and to bf16 one rounding of
2^-9. Losses are weighted means of log-probabilities: their absolute error times the weights' sum.
"""
import torch
import torch.nn.functional as F

REL = 1.5e-5
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -23}  # and the neighbour that a value near a tie takes


def counted(targets, vocab, ignore_index=-100):
    return (targets >= 0) & (targets < vocab) & (targets != ignore_index)


def token_logps(logits, targets, temperature=1.0, ignore_index=-100):
    """logits float64 [n, vocab], targets [n]; rows that do not count are 0 and have no gradient."""
    ok = counted(targets, logits.shape[-1], ignore_index)
    safe = torch.where(ok[:, None], logits, torch.zeros_like(logits))
    logp = F.log_softmax(safe / temperature, dim=-1).gather(1, torch.where(ok, targets, 0)[:, None]).squeeze(1)
    return torch.where(ok, logp, torch.zeros_like(logp))


def sequence_of(n, offsets):
    """Sequence of each row, -1 for none."""
    seq = torch.full((n,), -1, dtype=torch.long)
    for s in range(len(offsets) - 1):
        seq[offsets[s]:offsets[s + 1]] = s
    return seq


def preference(logits, targets, ref, offsets, beta, kind, smoothing=0.0, normalized=False, ignore_index=-100):
    ok = counted(targets, logits.shape[-1], ignore_index)
    gap = torch.where(ok, token_logps(logits, targets, 1.0, ignore_index) - ref.double(), 0.0)
    d = []
    for a, b in zip(offsets, offsets[1:]):
        x = gap[a:b].sum()
        d.append(x / max(1, int(ok[a:b].sum())) if normalized else x)
    pairs = len(d) // 2
    if pairs == 0:
        return logits.sum() * 0, torch.zeros(0).double(), torch.zeros(0).double()
    d = torch.stack(d)
    h = d[:pairs] - d[pairs:]
    if kind == "sigmoid":
        each = -(1 - smoothing) * F.logsigmoid(beta * h) - smoothing * F.logsigmoid(-beta * h)
    elif kind == "ipo":
        each = (h - 1 / (2 * beta)) ** 2
    else:
        each = torch.relu(1 - beta * h)
    return each.mean(), beta * d[:pairs], beta * d[pairs:]


def row_weights(ok, seq, reduction):
    """ok: rows that count; seq: their sequences."""
    ok = ok.double()
    if reduction == "sum":
        return ok
    if reduction in ("token", "mean"):
        return ok / max(1.0, float(ok.sum()))
    w = torch.zeros_like(ok)
    filled = [s for s in range(int(seq.max()) + 1 if seq.numel() else 0) if float(ok[seq == s].sum()) > 0]
    for s in filled:
        w[seq == s] = ok[seq == s] / ok[seq == s].sum() / len(filled)
    return w


def policy(logits, targets, old, adv_rows, ref, weight, ok, lo, hi, kl_coef, temperature, ignore_index=-100):
    """adv_rows, weight, ok: of the rows. Returns (loss, logps, (mean KL, clipped share))."""
    logp = token_logps(logits, targets, temperature, ignore_index)
    ratio = torch.exp(logp - old.double())
    free, held = ratio * adv_rows, ratio.clamp(1 - lo, 1 + hi) * adv_rows
    each = -torch.minimum(free, held)
    kl = torch.zeros_like(each)
    if ref is not None:
        delta = ref.double() - logp
        kl = torch.expm1(delta) - delta
        each = each + kl_coef * kl
    n = max(1, int(ok.sum()))
    stats = torch.stack([kl[ok].sum() / n, (free > held)[ok].double().sum() / n])
    return torch.where(ok, each * weight, 0.0).sum(), torch.where(ok, logp, 0.0), stats


def distill(logits, ids, teacher, lse, ok, weight, temperature):
    """ids [n, k] with -1 for entries left out, repeated ids adding up; ok, weight of the rows."""
    n, vocab = logits.shape
    total = logits.sum() * 0 if bool(torch.isfinite(logits).all()) else torch.zeros((), dtype=torch.float64)
    for r in range(n):
        if not bool(ok[r]):
            continue
        use = (ids[r] >= 0) & (ids[r] < vocab)
        t = teacher[r].double()[use] / temperature
        p_entry = torch.softmax(t, 0) if lse is None else torch.exp(t - lse[r].double())
        p = torch.zeros(vocab, dtype=torch.float64).index_add(0, ids[r][use], p_entry)
        where = torch.zeros(vocab, dtype=torch.bool)
        where[ids[r][use]] = True
        logq = F.log_softmax(logits[r] / temperature, dim=0)
        at = where & (p > 0)
        loss = (p[at] * (p[at].log() - logq[at])).sum()
        if lse is not None:
            left = 1 - p.sum()
            if left > 0:
                loss = loss + left * (left.log() - torch.logsumexp(logq[~where], 0))
        total = total + weight[r] * loss * temperature ** 2
    return total
