"""The losses over logits where a call is out of the ordinary: tensor subclasses among the arguments, hooks on what a
backward keeps, values past fp32 and NaN, sums that nearly cancel, no rows, as many rows as a launch holds and batches of
many; and the distillation loss at each width of the kernels that keep a row."""
import math

import pytest
import torch
import torch.utils.checkpoint

from micro_engram_fork_amd import _lib, losses

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROWS, VOCAB = (2, 3), 77


def _gen(seed):
    return torch.Generator().manual_seed(seed)


class _Wrapped(torch.Tensor):
    """A subclass that holds another tensor and hands every op that tensor."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

    def __init__(self, inner):
        self.inner = inner

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        res = func(*(a.inner if isinstance(a, cls) else a for a in args), **(kwargs or {}))
        # values made from a wrapped one are wrapped, results of this library's ops plain
        return cls(res) if func.namespace == "aten" and isinstance(res, torch.Tensor) else res


def _arguments():
    """name -> (function, its arguments but the logits)."""
    values = lambda seed, *shape: torch.randn(*shape, generator=_gen(seed)).to(DEV)  # noqa: E731
    targets = torch.randint(0, VOCAB, ROWS, generator=_gen(1)).to(DEV)
    ids = torch.stack([torch.randperm(VOCAB, generator=_gen(k))[:4] for k in range(6)]).view(*ROWS, 4).to(DEV)
    teacher = values(2, *ROWS, 4)
    cu = torch.tensor([0, 2, 6], device=DEV)
    return {
        "token_logps": (losses.token_logps, dict(targets=targets)),
        "preference": (losses.preference_loss, dict(targets=targets, ref_logps=values(3, *ROWS) - 4, cu_seqlens=cu)),
        "policy": (losses.policy_loss, dict(targets=targets, old_logps=values(4, *ROWS) - 4, advantages=values(5, 2),
                                            ref_logps=values(6, *ROWS) - 4, cu_seqlens=cu, kl_coef=0.3)),
        "distill": (losses.distill_loss, dict(teacher_ids=ids, teacher_logits=teacher, teacher_lse=teacher.logsumexp(-1) + 0.3,
                                              mask=torch.tensor([[True, True, False], [True, False, True]], device=DEV))),
    }


def _first(out):
    return out[0] if isinstance(out, tuple) else out


@pytest.mark.parametrize("name,wrapped", [
    ("token_logps", "targets"), ("preference", "ref_logps"), ("preference", "cu_seqlens"), ("policy", "old_logps"),
    ("policy", "advantages"), ("policy", "ref_logps"), ("policy", "cu_seqlens"), ("distill", "teacher_logits"),
    ("distill", "teacher_lse"), ("distill", "mask"), ("distill", "upstream"), ("policy", "upstream"), ("preference", "upstream"),
    ("token_logps", "upstream")])
def test_subclasses_give_the_values_of_what_they_hold(name, wrapped):
    fn, args = _arguments()[name]
    x = torch.randn(*ROWS, VOCAB, generator=_gen(9)).to(DEV).requires_grad_()
    want = _first(fn(x, **args))
    upstream = torch.full_like(want, 3.0)
    want_grad, = torch.autograd.grad(want, x, upstream)
    if wrapped == "upstream":
        upstream = _Wrapped(upstream)
    else:
        args[wrapped] = _Wrapped(args[wrapped])
    got = _first(fn(x, **args))
    grad, = torch.autograd.grad(got, x, upstream)
    # the same kernels on the same values
    assert torch.equal(got, want) and torch.equal(grad, want_grad)


# ------------------------------------------------------------------------------- saved tensors
WIDE = 1 << 20  # columns added to the logits, 24 MB in all


def _close(a, b):
    """Gradients of one row kernel and of two sweeps: probabilities off by 1.5e-5 of themselves in each."""
    torch.testing.assert_close(a, b, rtol=6e-5, atol=1e-9)


@pytest.mark.parametrize("name", ["token_logps", "preference", "policy", "distill"])
@pytest.mark.parametrize("way", ["save_on_cpu", "checkpoint"])
def test_what_saved_tensor_hooks_take_is_not_held_beside(name, way):
    fn, args = _arguments()[name]
    x = torch.randn(*ROWS, VOCAB, generator=_gen(9)).to(DEV).requires_grad_()
    wide = torch.full((*ROWS, WIDE), -1e4, device=DEV)

    def value(z):
        return _first(fn(torch.cat([z, wide], dim=-1), **args))

    plain = value(x)
    want, = torch.autograd.grad(plain.sum(), x)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    if way == "save_on_cpu":
        with torch.autograd.graph.save_on_cpu():
            loss = value(x)
    else:
        loss = torch.utils.checkpoint.checkpoint(value, x, use_reentrant=False)
    assert torch.cuda.memory_allocated() - before < 1 << 20  # the graph alone
    grad, = torch.autograd.grad(loss.sum(), x)
    assert torch.allclose(loss, plain, rtol=1e-5, atol=1e-6)
    _close(grad, want)


# -------------------------------------------------------------------------------------- policy
ROUTES = [(3, 7), (6, 640), (2, 9000)]  # rows and vocabulary: two sweeps, one read, rows in parts


def _sampled(n, vocab):
    """Logits that want gradients, targets, their log-probabilities as the losses give them."""
    x = torch.randn(n, vocab, generator=_gen(2)).to(DEV).requires_grad_()
    targets = torch.randint(0, vocab, (n,), generator=_gen(3)).to(DEV)
    return x, targets, losses.token_logps(x.detach(), targets)


@pytest.mark.parametrize("d", [1e-6, 1e-4, 3e-3, 0.02, 0.24, 0.26, 0.49, 0.51, 1.0, 5.0, 40.0])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_policy_kl_of_small_differences_keeps_its_digits(d, sign):
    # one token in all: its log-probability is 0 exactly, the difference the reference's. The value is a series of a few
    # terms or a difference that loses at most two bits: 1e-6 of itself
    ref = torch.tensor([sign * d], device=DEV)
    x = torch.randn(1, 1, generator=_gen(1)).to(DEV)
    loss, logps, stats = losses.policy_loss(x, torch.zeros(1, dtype=torch.long, device=DEV), torch.zeros(1, device=DEV),
                                            torch.zeros(1, device=DEV), ref_logps=ref, kl_coef=1.0)
    d = float(ref)
    want = math.expm1(d) - d if abs(d) > 1e-2 else sum(d ** k / math.factorial(k) for k in range(2, 9))
    assert float(logps) == 0.0
    assert float(stats[0]) == pytest.approx(want, rel=1e-6) and float(loss) == pytest.approx(want, rel=1e-6)


@pytest.mark.parametrize("n,vocab", ROUTES)
def test_policy_kl_of_a_token_ruled_out_is_infinite(n, vocab):
    x, targets, old = _sampled(n, vocab)
    x.data[1, targets[1]] = -float("inf")
    for kl_coef in (0.0, 0.1):
        stats = losses.policy_loss(x.detach(), targets, old, torch.ones(n, device=DEV), ref_logps=old, kl_coef=kl_coef)[2]
        assert float(stats[0]) == float("inf")


@pytest.mark.parametrize("n,vocab", ROUTES)
@pytest.mark.parametrize("far", ["reference", "logit"])
def test_policy_with_the_kl_as_a_statistic_alone(n, vocab, far):
    # kl_coef 0: no KL term, also where its value is past fp32
    x, targets, old = _sampled(n, vocab)
    ref = old.clone()
    if far == "reference":
        ref[1] += 100.0
    else:  # a token that has been ruled out since it was sampled
        x.data[1, targets[1]] = -float("inf")
    adv = torch.tensor([2.0, 0.5, -1.0, 1.0, 1.0, 3.0], device=DEV)[:n]
    want, _, _ = losses.policy_loss(x, targets, old, adv)
    want_grad, = torch.autograd.grad(want, x)
    loss, _, stats = losses.policy_loss(x, targets, old, adv, ref_logps=ref, kl_coef=0.0)
    grad, = torch.autograd.grad(loss, x)
    assert bool(want.isfinite()) and torch.equal(loss, want) and torch.equal(grad, want_grad)
    assert float(stats[0]) == float("inf")
    with torch.no_grad():
        assert bool(losses.policy_loss(x, targets, old, adv, ref_logps=ref)[0].isfinite())


@pytest.mark.parametrize("n,vocab", ROUTES)
def test_policy_of_an_advantage_of_zero(n, vocab):
    # its term is 0 at any ratio, also one past fp32; a ratio that is NaN stays NaN
    x, targets, old = _sampled(n, vocab)
    old[1] = -200.0
    adv = torch.ones(n, device=DEV)
    adv[1] = 0.0
    loss, _, stats = losses.policy_loss(x, targets, old, adv, reduction="sum")
    grad, = torch.autograd.grad(loss, x)
    # ratios of 1 up to the rounding of log-probabilities in other orders of the sum
    assert float(loss) == pytest.approx(1.0 - n, abs=(n - 1) * 1.5e-5)
    assert int(grad[1].count_nonzero()) == 0 and bool(grad.isfinite().all()) and float(stats[1]) == 0.0
    with torch.no_grad():
        assert float(losses.policy_loss(x, targets, old, adv, reduction="sum")[0]) == pytest.approx(1.0 - n, abs=(n - 1) * 1.5e-5)
    old[1] = float("nan")
    assert bool(losses.policy_loss(x, targets, old, adv)[0].isnan())


# ---------------------------------------------------------------------------------- preference
def _pair_of_sums(chosen, rejected, normalized, kind, beta):
    """preference_loss of two sequences whose differences to the reference are given (one token in all: log-probabilities
    of 0 exactly), and its 64-bit value."""
    ref = -torch.tensor([*chosen, *rejected], dtype=torch.float32)
    n = len(ref)
    cu = torch.tensor([0, len(chosen), n], device=DEV)
    got = losses.preference_loss(torch.zeros(n, 1, device=DEV), torch.zeros(n, dtype=torch.long, device=DEV), ref.to(DEV),
                                 cu_seqlens=cu, beta=beta, loss_type=kind, length_normalized=normalized)
    d = [float((-part.double()).sum()) / (len(part) if normalized else 1) for part in ref.split([len(chosen), len(rejected)])]
    h = d[0] - d[1]
    want = {"sigmoid": math.log1p(math.exp(-abs(beta * h))) + max(-beta * h, 0.0), "ipo": (h - 0.5 / beta) ** 2,
            "hinge": max(0.0, 1 - beta * h)}[kind]
    return got, want, d


@pytest.mark.parametrize("kind", ["sigmoid", "ipo", "hinge"])
@pytest.mark.parametrize("normalized", [False, True])
def test_preference_of_long_answers_far_from_the_reference(kind, normalized):
    # sums of about 5000 (means of about 1) that differ by little: h keeps the digits that each has past fp32
    g = _gen(4)
    base = torch.rand(5000, generator=g) + 0.5
    chosen, rejected = (base + 1e-4).tolist(), base[torch.randperm(5000, generator=g)].tolist()
    beta = 0.5 if not normalized else 50.0
    got, want, d = _pair_of_sums(chosen, rejected, normalized, kind, beta)
    # h is exact up to its own rounding; a few roundings of fp32 follow
    assert float(got[0]) == pytest.approx(want, rel=1e-6)
    assert float(got[1]) == pytest.approx(beta * d[0], rel=3e-7) and float(got[2]) == pytest.approx(beta * d[1], rel=3e-7)


@pytest.mark.parametrize("smoothing", [0.0, 1.0])
@pytest.mark.parametrize("side", [0, 1])
def test_preference_of_an_answer_that_cannot_be(side, smoothing):
    # a token of it is ruled out: its sum is minus infinity. The sigmoid loss is 0 where that is as it should be, and
    # infinite where not, whose gradient is that of an ordinary lost pair
    n, vocab = 6, 50
    x = torch.randn(n, vocab, generator=_gen(5))
    targets = torch.arange(n)
    x[3 * side + 1, targets[3 * side + 1]] = -float("inf")
    xg = x.to(DEV).requires_grad_()
    loss, chosen, rejected = losses.preference_loss(xg, targets.to(DEV), torch.zeros(n, device=DEV),
                                                    cu_seqlens=torch.tensor([0, 3, 6], device=DEV), beta=0.5, label_smoothing=smoothing)
    grad, = torch.autograd.grad(loss, xg)
    assert float((chosen, rejected)[side]) == -float("inf") and bool((chosen, rejected)[1 - side].isfinite().all())
    wanted = side == (1 if smoothing == 0.0 else 0)  # the answer that should lose
    assert float(loss) == (0.0 if wanted else float("inf"))
    assert bool(grad.isfinite().all())
    q = torch.softmax(x.double(), -1)
    c = torch.tensor([1.0, -1.0]).repeat_interleave(3)[:, None] * (0.5 if smoothing else -0.5)
    want = c * (torch.nn.functional.one_hot(targets, vocab) - q) * (0.0 if wanted else 1.0)
    torch.testing.assert_close(grad.double().cpu(), want, rtol=3e-5, atol=1e-9)


# -------------------------------------------------------------------------------------- no rows
@pytest.mark.parametrize("shape", [(2, 3, 0, 10), (2, 0, 3, 10)])
def test_no_rows_in_many_dims(shape):
    x = torch.zeros(shape, device=DEV, requires_grad=True)
    targets, rows = torch.zeros(shape[:-1], dtype=torch.long, device=DEV), torch.zeros(shape[:-1], device=DEV)
    pairs = math.prod(shape[:-2]) // 2
    out = losses.token_logps(x, targets)
    assert out.shape == targets.shape and torch.autograd.grad(out.sum(), x)[0].shape == x.shape
    loss, chosen, _ = losses.preference_loss(x, targets, rows)
    assert float(loss.detach()) == pytest.approx(math.log(2) if pairs else 0.0) and chosen.tolist() == [0.0] * pairs
    assert torch.autograd.grad(loss, x)[0].shape == x.shape
    for loss in (losses.policy_loss(x, targets, rows, rows)[0], losses.distill_loss(x, targets[..., None], rows[..., None])):
        assert float(loss.detach()) == 0 and torch.autograd.grad(loss, x)[0].shape == x.shape


# ------------------------------------------------------------------------------------ most rows
MOST_SHORT = (2 ** 32 - 1) // 64 - 16  # rows of up to 2048 tokens that a launch holds


def test_as_many_rows_as_a_launch_holds():
    # one row in memory, expanded; targets that differ at both ends and in the middle
    n, vocab = MOST_SHORT, 8
    row = torch.randn(vocab, generator=_gen(6)).bfloat16().to(DEV)
    targets = torch.zeros(n, dtype=torch.int32, device=DEV)
    for r in (0, n // 2, n - 1):
        targets[r] = 5
    x = row.expand(n, vocab).requires_grad_()
    out = losses.token_logps(x, targets)
    grad, = torch.autograd.grad(out, x, torch.ones(n, device=DEV))
    want = torch.log_softmax(row.double(), -1)
    for t, count in ((5, 3), (0, n - 3)):
        here = targets == t
        value = out[here]
        assert int(here.sum()) == count and bool((value == value[0]).all())
        assert float(value[0]) == pytest.approx(float(want[t]), abs=1.5e-5)
        rows = grad[here]
        assert bool((rows == rows[0]).all())
        g = torch.nn.functional.one_hot(torch.tensor(t), vocab).to(DEV) - want.exp()
        torch.testing.assert_close(rows[0].double(), g, rtol=2.0 ** -8, atol=1.5e-5)


def test_more_rows_are_refused():
    n, vocab = MOST_SHORT + 1, 8
    x = torch.zeros(vocab, device=DEV).expand(n, vocab)
    with pytest.raises(_lib.EngramLibError, match="too many rows"):
        losses.token_logps(x, torch.zeros(n, dtype=torch.int32, device=DEV))


# -------------------------------------------------------------------------------- distillation
# one width of each kernel that keeps rows, as (dtype, vocabulary): 64, 256, 512 and 1024 threads, 22 units in
# registers, with LDS, with a second read
DISTILL_WIDTHS = [(torch.bfloat16, v) for v in (64, 1000, 8201, 40_001, 70_003, 140_001, 262_144, 300_007)] + \
                 [(torch.float32, v) for v in (64, 4099, 16_391, 40_003, 70_001, 131_072)]


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype,vocab", DISTILL_WIDTHS)
def test_distillation_loss_of_each_row_width(dtype, vocab, rest):
    rows, top, temp, scale = 260, 5 if vocab < 100 else 70, 1.5, 0.5
    g = torch.Generator(device=DEV).manual_seed(vocab)
    x = torch.randn(rows, vocab, generator=g, device=DEV) * 2
    start = torch.randint(0, vocab, (rows, 1), generator=g, device=DEV)
    ids = (start + torch.randint(1, vocab // top + 1, (rows, top), generator=g, device=DEV).cumsum(1)) % vocab
    x.scatter_(1, ids[:, :1], math.log(vocab) + 1.0)
    x = x.to(dtype)
    ids[3, 2:4] = ids[3, 0]  # entries of one token
    ids[4, 1:] = -1
    ids[5] = -1              # does not count
    mask = torch.ones(rows, dtype=torch.bool, device=DEV)
    mask[30:60:2] = False
    x[9, ids[9, 0]] = -float("inf")  # a token that the teacher wants and the student rules out
    teacher = (torch.randn(rows, top, generator=g, device=DEV) * 2 + 10).to(dtype)
    use = ids >= 0
    t64 = torch.where(use, teacher.double() / temp, -float("inf"))
    lse = (t64.logsumexp(1) + 0.1 + 0.2 * torch.rand(rows, generator=g, device=DEV)).nan_to_num(0, 0, 0).float() if rest else None
    ok = mask & use.any(1)
    # the definition in 64 bits, a token's entries added up
    p_entry = torch.where(use, (t64 - (t64.logsumexp(1, keepdim=True) if lse is None else lse[:, None].double())).exp(), 0.0)
    p = torch.zeros(rows, vocab, dtype=torch.float64, device=DEV).scatter_add_(1, ids.clamp(min=0), p_entry)
    where = torch.zeros(rows, vocab, device=DEV).scatter_add_(1, ids.clamp(min=0), use.float()) > 0
    logq = torch.log_softmax(x.double() / temp, -1)
    each = torch.where(p > 0, p * (p.clamp(min=1e-300).log() - logq), 0.0).sum(1)
    size = torch.where(p > 0, p * logq.abs(), 0.0).sum(1)
    if rest:
        left, other = 1 - p.sum(1), torch.where(where, -float("inf"), logq).logsumexp(1)
        each, size = each + left * (left.log() - other), size + left * (left.log() - other).abs()
    xg = x.clone().requires_grad_()

    def loss(counting):
        return losses.distill_loss(xg, ids, teacher, teacher_lse=lse, mask=counting, temperature=temp, scale=scale)

    assert float(loss(mask)) == float("inf")
    mask[9] = ok[9] = False
    want = float(scale * temp ** 2 * each[ok].mean())
    # log q and log p are off by 1.5e-5 each, with the rest class its logarithm too, and by the rounding of themselves
    tol = scale * temp ** 2 * (3 * 1.5e-5 + 4e-7 * float(size[ok].mean())) + 1e-6 * abs(want)
    assert float(loss(mask)) == pytest.approx(want, abs=tol)
    with torch.no_grad():
        assert float(loss(mask)) == pytest.approx(want, abs=tol)


# ------------------------------------------------------------------------------------ many rows
MANY = 70_001


def _many(vocab):
    """Rows of a small vocabulary on the GPU with targets, a few that do not count, and their log-probabilities in 64 bits."""
    g = torch.Generator(device=DEV).manual_seed(vocab)
    x = torch.randn(MANY, vocab, generator=g, device=DEV) * 2
    targets = torch.randint(0, vocab, (MANY,), generator=g, device=DEV)
    targets[torch.rand(MANY, generator=g, device=DEV) < 0.2] = -100
    ok = targets >= 0
    now = torch.log_softmax(x.double(), -1).gather(1, targets.clamp(min=0)[:, None]).squeeze(1)
    return x, targets, ok, torch.where(ok, now, 0.0), g


def _row_grad(x, targets, coef):
    g = -coef[:, None] * torch.softmax(x.double(), -1)
    return g.scatter_add(1, targets.clamp(min=0)[:, None], coef[:, None])


def _close_rows(grad, want, coef):
    tol = 6e-5 * coef.abs()[:, None] + 2.0 ** -23 * want.abs() + 1e-37
    assert bool(((grad.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("vocab", [9, 70])  # two sweeps, one read
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_policy_of_many_rows_in_sequences_of_all_lengths(vocab, reduction):
    x, targets, ok, now, g = _many(vocab)
    cu = torch.tensor([0, 1, 1, 40_000, 40_003, 69_000, 70_000], device=DEV)  # the last row is of no sequence
    seqs = len(cu) - 1
    seq = torch.bucketize(torch.arange(MANY, device=DEV), cu[1:], right=True)
    adv = torch.randn(seqs, generator=g, device=DEV)
    old = (now - 0.1 * torch.rand(MANY, generator=g, device=DEV)).float()
    counts = ok & (seq < seqs)
    lengths = torch.zeros(seqs + 1, dtype=torch.float64, device=DEV).index_add(0, seq, counts.double())[:seqs]
    weight = counts.double() / counts.sum()
    if reduction == "sequence":
        weight = counts / lengths.clamp(min=1)[seq.clamp(max=seqs - 1)] / (lengths > 0).sum()
    adv_rows = adv.double()[seq.clamp(max=seqs - 1)]
    ratio = torch.exp(now - old.double())  # 1 to 1.11: inside the bounds
    xg = x.clone().requires_grad_()
    loss, logps, stats = losses.policy_loss(xg, targets, old, adv[:, None], cu_seqlens=cu, reduction=reduction)
    grad, = torch.autograd.grad(loss, xg)
    want = -(ratio * adv_rows * weight).sum()
    # a ratio has the error of its log-probability, 1.5e-5, and the roundings of itself and of a weight
    size = float((ratio * adv_rows.abs() * weight).sum())
    assert float(loss) == pytest.approx(float(want), abs=2e-5 * size)
    assert bool(((logps.double() - now).abs()[counts] <= 1.5e-5 + 1e-6 * now.abs()[counts]).all())
    coef = -ratio * adv_rows * weight
    _close_rows(grad, _row_grad(x, targets, coef), coef)
    assert int(grad[~counts].count_nonzero()) == 0 and stats.tolist() == [0.0, 0.0]


@pytest.mark.parametrize("vocab", [9, 70])
def test_distillation_of_many_rows(vocab):
    x, targets, _, _, g = _many(vocab)
    mask = targets >= 0
    ids = torch.randint(0, vocab, (MANY, 1), generator=g, device=DEV)
    xg = x.clone().requires_grad_()
    loss = losses.distill_loss(xg, ids, torch.zeros(MANY, 1, device=DEV), mask=mask)
    grad, = torch.autograd.grad(loss, xg)
    # one entry has all of the teacher: minus its log-probability
    each = -torch.log_softmax(x.double(), -1).gather(1, ids).squeeze(1)
    want = each[mask].mean()
    assert float(loss) == pytest.approx(float(want), abs=2 * 1.5e-5 + 1e-6 * float(want))
    coef = -mask.double() / mask.sum()
    _close_rows(grad, _row_grad(x, ids.squeeze(1), coef), coef)


@pytest.mark.parametrize("vocab", [9, 70])
def test_preference_of_many_pairs(vocab):
    x, targets, ok, now, g = _many(vocab)
    pairs = 10_000
    cuts = torch.sort(torch.randint(0, MANY, (2 * pairs - 1,), generator=g, device=DEV)).values
    cu = torch.cat([torch.tensor([0], device=DEV), cuts, torch.tensor([MANY], device=DEV)])
    ref = (now + 0.1 * torch.randn(MANY, generator=g, device=DEV)).float()
    seq = torch.bucketize(torch.arange(MANY, device=DEV), cu[1:], right=True)
    d = torch.zeros(2 * pairs, dtype=torch.float64, device=DEV).index_add(0, seq, torch.where(ok, now - ref.double(), 0.0))
    longest = int(torch.bincount(seq).max())
    xg = x.clone().requires_grad_()
    loss, chosen, rejected = losses.preference_loss(xg, targets, ref, cu_seqlens=cu, beta=0.5)
    grad, = torch.autograd.grad(loss, xg)
    h = d[:pairs] - d[pairs:]
    off = 1.5e-5 * longest + 3e-7 * float(d.abs().max())  # log-probabilities off by 1.5e-5 each
    assert float(loss) == pytest.approx(float(torch.nn.functional.softplus(-0.5 * h).mean()), abs=2 * 0.5 * off)
    got = torch.cat([chosen, rejected]).double()
    assert bool(((got - 0.5 * d).abs() <= 0.5 * off).all())
    slope = -0.5 * torch.sigmoid(-0.5 * h) / pairs
    coef = torch.where(ok, torch.cat([slope, -slope])[seq], 0.0)
    want = _row_grad(x, targets, coef)
    # the factor's derivative by h is at most 1/4 of 0.5^2 / pairs
    tol = 6e-5 * coef.abs()[:, None] + 2 * off * 0.0625 / pairs + 2.0 ** -23 * want.abs()
    assert bool(((grad.double() - want).abs() <= tol).all()) and int(grad[~ok].count_nonzero()) == 0


def test_policy_of_no_sequences():
    # rows, but no sequence that holds one, and so no advantage either
    x = torch.randn(5, 33, generator=_gen(7)).to(DEV).requires_grad_()
    rows, targets = torch.zeros(5, device=DEV), torch.zeros(5, dtype=torch.long, device=DEV)
    for reduction in ("token", "sequence", "sum"):
        loss, logps, stats = losses.policy_loss(x, targets, rows, torch.zeros(0, device=DEV), reduction=reduction,
                                                cu_seqlens=torch.zeros(1, dtype=torch.long, device=DEV))
        grad, = torch.autograd.grad(loss, x)
        assert float(loss.detach()) == 0 and logps.tolist() == [0.0] * 5 and stats.tolist() == [0.0, 0.0]
        assert int(grad.count_nonzero()) == 0


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,vocab", ROUTES)
def test_distillation_of_a_logit_that_is_none(n, vocab, dtype, rest):
    # among the teacher's entries or the other tokens: the row has no loss, whatever the entry's own probability
    top = min(5, vocab - 1)
    ids = torch.stack([torch.randperm(vocab, generator=_gen(k))[:top] for k in range(n)]).to(DEV)
    teacher = torch.randn(n, top, generator=_gen(8)).to(DEV)
    teacher[:, 1] = -200.0  # an entry of probability 0
    lse = teacher.logsumexp(-1) + 0.3 if rest else None
    base = torch.randn(n, vocab, generator=_gen(9)).to(dtype).to(DEV)
    others = [j for j in range(vocab) if j not in ids[1].tolist()]
    for token in (int(ids[1, 0]), int(ids[1, 1]), int(ids[1, top - 1]), others[0], others[-1]):
        x = base.clone()
        x[1, token] = float("nan")
        xg = x.requires_grad_()
        loss = losses.distill_loss(xg, ids, teacher, teacher_lse=lse)
        grad, = torch.autograd.grad(loss, xg)
        assert bool(loss.isnan()) and bool(grad[1].isnan().any()) and bool(grad[0].isfinite().all()), token
        with torch.no_grad():
            assert bool(losses.distill_loss(xg, ids, teacher, teacher_lse=lse).isnan())
