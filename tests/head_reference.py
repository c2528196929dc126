"""The losses over a decoder's head in float64, with bounds on what the kernels' arithmetic may be off by.

Bounds, from the arithmetic. A logit is a sum of dim products accumulated in fp32 (at most dim roundings, each of at
most 2^-24 of the sum of the products' sizes so far; fp32 operands as bf16 parts: six sums, and products left
out under 2^-24): dz = (dim + 8) 2^-24 sum |h w| / T, three times that for fp32. Statistics are sums of positive
terms in fp32: their logs are off by dz and by 2e-6 (fewer than 16 roundings in a row of each tree, exponentials of
2 ulp). A value of the gradient dz_ij is off relatively by twice that (its exponent and its sum) and by 1e-6 of its
roundings, to which bf16 adds 2^-8: not at a row's target for the gradient of the hidden states, and up to 128 rows
(counted or not) only 2^-16 for that of the head; its products with W or h are accumulated in fp32, and the result is
rounded to its type (half a step: 2^-8 or 2^-24). Exponentials and bf16 parts under 2^-126, the smallest normal number,
may be taken as zeros: 2^-126 more for q, times the row's factor, and for the value of the gradient itself."""
import torch


def counted(targets, vocab, ignore_index=-100):
    return (targets >= 0) & (targets < vocab) & (targets != ignore_index)


def head(hidden, weight, targets, dtype, temperature=1.0, ignore_index=-100, upstream=None, smoothing=0.0, z_loss=0.0,
         scale=1.0, mean=True):
    """hidden [n, dim], weight, targets [n] (values that the kernels get, any float type). upstream: [n] for
    log-probabilities, or None for the cross entropy with an upstream gradient of 1. A dict of
    name -> (float64 value, bound): "logps" or "loss", "hidden", "weight"."""
    vocab, dim = weight.shape
    ok = counted(targets, vocab, ignore_index)
    h, w = hidden[ok].double(), weight.double()
    t = targets[ok].long()
    n = h.shape[0]
    wide = dtype is torch.float32
    z = h @ w.t() / temperature
    dz = (3 if wide else 1) * (dim + 8) * 2.0 ** -24 * (h.abs() @ w.abs().t()) / temperature
    dmax = dz.amax(1) if n else torch.zeros(0, dtype=torch.float64, device=h.device)
    lse = torch.logsumexp(z, 1) if n else dmax
    rows = torch.arange(n, device=h.device)
    logp = z[rows, t] - lse
    dlog = 2 * dmax + 2e-6 + 2.0 ** -22 * (lse.abs() + z[rows, t].abs())
    out = {}

    def full(x):
        res = torch.zeros(targets.shape[0], *x.shape[1:], dtype=torch.float64, device=h.device)
        res[ok] = x
        return res
    q = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(q)
    hot[rows, t] = 1.0
    if upstream is not None:
        out["logps"] = full(logp), full(dlog + 2.0 ** -22 * logp.abs())
        c = -upstream[ok].double() / temperature
        a, b = torch.ones_like(c), 0.0
        factor = torch.zeros_like(c)
    else:
        each = -logp + smoothing * (z[rows, t] - z.mean(1)) + z_loss * lse ** 2
        err = dlog * (1 + 2 * z_loss * lse.abs()) + 2 * smoothing * (dmax + 2.0 ** -20 * z.abs().mean(1)) + 2.0 ** -21 * each.abs() + 2.0 ** -20 * z_loss * lse ** 2
        c = torch.full_like(lse, scale / ((max(n, 1) if mean else 1) * temperature))
        weighing = scale / (max(n, 1) if mean else 1)
        out["loss"] = each.sum() * weighing, (err.sum() * abs(weighing) + 2.0 ** -23 * abs(float(each.sum() * weighing)))
        a, b = 1 + 2 * z_loss * lse, smoothing / vocab
        factor = 2 * z_loss * (dlog + 2.0 ** -22 * lse.abs())
    g = a[:, None] * q - (1 - smoothing if upstream is None else 1.0) * hot - b
    # at the target the others' weight stands in place of the difference
    at = a * q[rows, t] - (1 - smoothing if upstream is None else 1.0) - b
    dg = a[:, None] * q * (2 * dz + dlog[:, None] + 1e-6) + factor[:, None] * q + 2.0 ** -22 * b
    others = 1 - q[rows, t]
    extra = (a - 1).abs() + (smoothing if upstream is None else 0.0) + b
    dg[rows, t] = a.abs() * (others * (2 * dmax + dlog + 1e-6)) + factor + 2.0 ** -22 * (extra + at.abs())
    half = 2.0 ** -24 if wide else 2.0 ** -8
    rounded = {"hidden": g.abs() * half, "weight": g.abs() * (half if targets.shape[0] > 128 else half * half)}
    rounded["hidden"][rows, t] = 0.0
    g, dg = g * c[:, None], (dg + g.abs() * 2.0 ** -22) * c.abs()[:, None]
    dg = dg + 2.0 ** -126 * (1 + (a * c).abs()[:, None])
    for name, value, x, y, k in (("hidden", g @ w, g.abs(), w.abs(), vocab), ("weight", g.t() @ h, g.abs().t(), h.abs(), n)):
        d = dg if wide else dg + rounded[name] * c.abs()[:, None]
        d = d if name == "hidden" else d.t()
        err = d @ y + (3 if wide else 1) * (k + 8) * 2.0 ** -24 * (x @ y) + half * (value.abs() + d @ y) + 2.0 ** -133
        out[name] = (full(value), full(err)) if name == "hidden" else (value, err)
    return out
