"""policy_loss and distill_loss where they write the gradient from one read of the logits (csrc/loss_rows.hip: batches of
many rows), at each of its row widths: rows shorter and longer than what registers, LDS and a second read hold,
against float64 on the GPU. Tolerances as in loss_reference.py."""
import math

import pytest
import torch

import loss_reference as ref64
from loss_reference import HALF_ULP, REL
from micro_engram_fork_amd import losses

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROWS = 260
# (dtype, vocab): both sides of each kernel's width, odd ones, one with a second read
WIDTHS = [(torch.bfloat16, v) for v in (64, 71, 1000, 8192, 8201, 32_768, 32_777, 131_072, 131_085, 250_001, 262_144, 300_007)] + \
         [(torch.float32, v) for v in (64, 515, 4096, 4099, 16_384, 16_391, 65_536, 65_543, 110_003, 131_072)]


def _rows(vocab, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(ROWS, vocab, generator=g, device=DEV) * 2
    hot = torch.randint(0, vocab, (ROWS, 1), generator=g, device=DEV)
    hot[0], hot[1], hot[2] = 0, vocab - 1, vocab // 8 * 8 - 1
    x.scatter_(1, hot, math.log(vocab) + 2 + torch.randn(ROWS, 1, generator=g, device=DEV))
    x = x.to(dtype)
    # rows whose own token is no guide to the row's sum, and rows at the ends of the type's range
    x[5, hot[5]] = -float("inf")
    x[6, hot[6]] = -300.0
    x[7] = torch.finfo(dtype).min
    x[8] = torch.finfo(dtype).max
    x[9, : vocab // 2] = -float("inf")
    x[10] += 5000.0
    return x, hot.squeeze(1), g


def _close(got, want, tol, what):
    got, want = got.detach().double(), want.detach().double()
    bad = ~((got - want).abs() <= tol) & ~(got.isnan() & want.isnan()) & ~(got == want)
    assert not bool(bad.any()), f"{what}: off by {float((got - want).abs()[bad].max()):.3g}, {int(bad.sum())} values in rows " \
                                f"{bad.nonzero()[:5].tolist()}"


@pytest.mark.parametrize("dtype,vocab", WIDTHS)
def test_policy_rows(dtype, vocab):
    x, targets, g = _rows(vocab, dtype, vocab)
    targets[11:40:3] = -100
    x[11] = float("nan")
    ok = ref64.counted(targets, vocab)
    logq = torch.where(ok[:, None], x.double(), 0.0).log_softmax(-1)
    q = logq.exp()
    now = torch.where(ok, logq.gather(1, targets.clamp(min=0)[:, None]).squeeze(1), 0.0)
    old = (now + 0.3 * torch.randn(ROWS, generator=g, device=DEV)).float()
    ref = (now + 0.2 * torch.randn(ROWS, generator=g, device=DEV)).float()
    adv = torch.randn(ROWS, generator=g, device=DEV)
    ref[5] = old[5] = -float("inf")  # its log-probability: ratio and KL are NaN there, by the definition
    lo, hi, kl = 0.2, 0.25, 0.1
    near = ((torch.exp(now - old.double()) - (1 - lo)).abs() < 1e-3) | ((torch.exp(now - old.double()) - (1 + hi)).abs() < 1e-3)
    old[near] += 0.01
    weight = ok.double() / ok.sum()
    leaf = torch.where(ok[:, None], x.double(), 0.0).requires_grad_()
    keep = torch.ones(ROWS, dtype=torch.bool, device=DEV)
    keep[5] = False  # left out of the sums' comparison
    logp = torch.where(ok, torch.log_softmax(leaf, -1).gather(1, targets.clamp(min=0)[:, None]).squeeze(1), 0.0)
    ratio = torch.exp(logp - old.double())
    free, held = ratio * adv, ratio.clamp(1 - lo, 1 + hi) * adv
    delta = ref.double() - logp
    each = -torch.minimum(free, held) + kl * (torch.expm1(delta) - delta)
    want_grad, = torch.autograd.grad((each * weight)[keep & ok].sum(), leaf)
    xg = x.clone().requires_grad_()
    loss, logps, stats = losses.policy_loss(xg, targets, old, adv, ref_logps=ref, kl_coef=kl, clip_low=lo, clip_high=hi)
    grad, = torch.autograd.grad(loss, xg)
    assert bool(loss.isnan()) and bool(grad[5].isnan().any())
    _close(logps[keep], logp[keep], REL + 1e-6 * logp.detach()[keep].abs(), "logps")
    coef = (ratio.detach().abs() * adv.abs() + kl * (1 + torch.exp(delta.detach()))) * weight
    base = q.scatter_add(1, targets.clamp(min=0)[:, None], torch.ones(ROWS, 1, dtype=torch.float64, device=DEV))
    tol = 4 * coef[:, None] * base * REL + want_grad.abs() * HALF_ULP[dtype] * 2 + 1e-37
    _close(grad[keep], want_grad[keep], tol[keep], "grad")
    assert int(grad[~ok].count_nonzero()) == 0
    # without the row that is NaN, the loss too; and an upstream gradient other than 1
    targets[5] = -100
    loss, _, stats = losses.policy_loss(xg, targets, old, adv, ref_logps=ref, kl_coef=kl, clip_low=lo, clip_high=hi, scale=0.5)
    n = int(ok.sum()) - 1
    want = (torch.where(ok & keep, each, 0.0).sum() / n).detach()
    _close(loss, want / 2, 4 * REL * float(torch.where(ok & keep, coef, 0.0).sum()) + 1e-6 * float(want.abs()) + 1e-8, "loss")
    tripled, = torch.autograd.grad(loss, xg, torch.tensor(3.0, device=DEV))
    again = losses.policy_loss(xg, targets, old, adv, ref_logps=ref, kl_coef=kl, clip_low=lo, clip_high=hi, scale=1.5)[0]
    direct, = torch.autograd.grad(again, xg)
    _close(tripled, direct.double(), direct.double().abs() * HALF_ULP[dtype] * 2 + 4 * 1.5 * tol / 4 + 1e-37, "upstream of 3")


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype,vocab", WIDTHS)
def test_distill_rows(dtype, vocab, rest):
    x, hot, g = _rows(vocab, dtype, vocab + 1)
    top = 5 if vocab < 100 else 70
    start = torch.randint(0, vocab, (ROWS, 1), generator=g, device=DEV)
    ids = (start + torch.randint(1, vocab // top + 1, (ROWS, top), generator=g, device=DEV).cumsum(1)) % vocab
    ids[:5, 0] = hot[:5]
    ids[0, 1], ids[1, 1], ids[2, 1] = vocab - 1, vocab - 2, 1  # the row's ends, and two entries in one chunk
    ids[3, 2:4] = ids[3, 0]  # entries of one token
    ids[4, 1:] = -1
    ids[12] = -1  # no entry at all: does not count
    x[8] = 1.0  # the type's largest everywhere: exponents of its differences alone; as ordinary values here
    teacher = (torch.randn(ROWS, top, generator=g, device=DEV) * 2 + 10).to(dtype)
    teacher[20, 0] = -float("inf")
    mask = torch.ones(ROWS, dtype=torch.bool, device=DEV)
    mask[30:60:2] = False
    x[30] = float("nan")
    temp = 1.5
    lse = None
    use = ids >= 0
    t64 = torch.where(use, teacher.double() / temp, -float("inf"))
    if rest:
        lse = (t64.logsumexp(1) + 0.1 + 0.2 * torch.rand(ROWS, generator=g, device=DEV)).nan_to_num(0, 0, 0).float()
    ok = mask & use.any(1)
    p_entry = torch.where(use, (t64 - (t64.logsumexp(1, keepdim=True) if lse is None else lse[:, None].double())).exp(), 0.0)
    p = torch.zeros(ROWS, vocab, dtype=torch.float64, device=DEV).scatter_add_(1, ids.clamp(min=0), p_entry)
    where = torch.zeros(ROWS, vocab, dtype=torch.bool, device=DEV)
    for i in range(top):
        at = use[:, i].nonzero().squeeze(1)
        where[at, ids[at, i]] = True
    leaf = torch.where(ok[:, None], x.double(), 0.0).requires_grad_()
    logq = torch.log_softmax(leaf / temp, -1)
    each = torch.where(p > 0, p * (p.clamp(min=1e-300).log() - logq), 0.0).sum(1)
    left = other = None
    if rest:
        left = 1 - p.sum(1)
        other = torch.where(where, -float("inf"), logq).logsumexp(1)
        each = each + left * (left.log() - other)
    finite = torch.isfinite(each) & ok
    weight = ok.double() / ok.sum()
    want = temp ** 2 * (each * weight)[finite].sum()
    want_grad, = torch.autograd.grad(want, leaf)
    xg = x.clone().requires_grad_()
    got = losses.distill_loss(xg, ids, teacher, teacher_lse=lse, mask=mask, temperature=temp)
    grad, = torch.autograd.grad(got, xg)
    # log q is off by REL and, where it is far below 0, by the rounding of itself
    tol = temp ** 2 * ((3 * REL + 4e-7 * torch.where(p > 0, p * logq.detach().abs().nan_to_num(0, 0, 0), 0.0).sum(1)) * weight)[finite].sum()
    if bool((finite == ok).all()):
        _close(got, want, float(tol) + 1e-6 * float(want.abs()), "loss")
    q = logq.detach().exp()
    share = 1 + (1 / torch.where(where, 0.0, q).sum(1, keepdim=True).clamp(min=1e-300) if rest else 0.0)
    tol = weight[:, None] * temp * (torch.where(where, q, q * share) * 3 + 2 * p) * REL + want_grad.abs() * HALF_ULP[dtype] + 1e-37
    _close(grad[finite], want_grad[finite], tol[finite], "grad")
    assert int(grad[~ok].count_nonzero()) == 0
    tripled, = torch.autograd.grad(losses.distill_loss(xg, ids, teacher, teacher_lse=lse, mask=mask, temperature=temp), xg,
                                   torch.tensor(3.0, device=DEV))
    _close(tripled[finite], 3 * want_grad[finite], 3 * tol[finite], "upstream of 3")


def test_same_bits_every_time():
    x, targets, g = _rows(262_144, torch.bfloat16, 1)
    targets[5] = -100
    old = torch.full((ROWS,), -2.0, device=DEV)
    adv = torch.randn(ROWS, generator=g, device=DEV)
    want = None
    for _ in range(3):
        xg = x.clone().requires_grad_()
        loss, logps, stats = losses.policy_loss(xg, targets, old, adv)
        grad, = torch.autograd.grad(loss, xg)
        if want is None:
            want = loss.clone(), logps.clone(), stats.clone(), grad.clone()
        assert all(torch.equal(a, b) for a, b in zip(want, (loss, logps, stats, grad)))
