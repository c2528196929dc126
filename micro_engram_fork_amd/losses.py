"""Losses over a decoder's logits, for training an engram past plain next-token text: distillation
from a teacher's top logits, preference pairs, sampled answers with advantages, and the
log-probabilities of given tokens that the last two take from a reference or an earlier policy.
(The reference trains with cross-entropy alone, micro_engram/train/head.py:85-165; that is
-token_logps(logits, targets).mean() here.)

    from micro_engram_fork_amd import losses
    with torch.no_grad():                     # the same decoder without its engram's rows
        ref = losses.token_logps(base_logits, targets)
    loss, chosen, rejected = losses.preference_loss(logits, targets, ref)
    loss.backward()

Logits are [..., vocab], bf16 or fp32, on the GPU, in any strides whose last is 1 (logits[:, :-1]
and a padded vocabulary's logits[..., :vocab] are read where they lie). Row i's target is the token
that row i predicts. Rows whose target is `ignore_index` (or no token at all) do not count: they
are not read, and their gradient is zeros. All sums, log-probabilities and losses are fp32 or
fp64 inside, whatever the logits are.

distill_loss and policy_loss know a row's gradient as soon as they have read the row, so with
gradients they write it in the forward and keep it for the backward, for an upstream gradient of 1.
The backward looks (on the device) whether that held, and computes the gradient again from the
logits if not: give a factor such as 1 / accumulation steps as `scale`, where it costs nothing. Under
hooks on saved tensors (torch.autograd.graph.save_on_cpu, non-reentrant checkpointing) nothing is kept
that does not pass through the hooks, and the gradient is written in the backward.
"""
import functools
import math

import torch
from torch.autograd.function import once_differentiable

from . import loss_ops
from ._lib import (ME_PAIR_HINGE, ME_PAIR_IPO, ME_PAIR_SIGMOID, ME_REDUCE_MEAN, ME_REDUCE_SEQUENCE,
                   ME_REDUCE_SUM)

IGNORE_INDEX = -100
TOP_MAX = 1024  # teacher entries of a row

_PAIR_LOSSES = {"sigmoid": ME_PAIR_SIGMOID, "ipo": ME_PAIR_IPO, "hinge": ME_PAIR_HINGE}
_POLICY_REDUCTIONS = {"token": ME_REDUCE_MEAN, "sequence": ME_REDUCE_SEQUENCE, "sum": ME_REDUCE_SUM}
_DISTILL_REDUCTIONS = {"mean": ME_REDUCE_MEAN, "sum": ME_REDUCE_SUM}


# ------------------------------------------------------------------------------------ checks
def _check_logits(logits):
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"[micro_engram] logits must be [..., vocab], got {tuple(logits.shape)}")
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"[micro_engram] logits must be bf16 or fp32, got {logits.dtype}")


def _check_targets(logits, targets):
    _check_logits(logits)
    if targets.shape != logits.shape[:-1]:
        raise ValueError(f"[micro_engram] targets {tuple(targets.shape)} do not match the logits' rows "
                         f"{tuple(logits.shape[:-1])}")
    if targets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"[micro_engram] targets must be int32 or int64, got {targets.dtype}")


def _check_number(value, what, low=0.0, high=math.inf, open_low=False):
    if type(value) is float and low < value < high:
        return value
    value = float(value)
    if not (low < value if open_low else low <= value) or not value <= high or math.isinf(value):
        raise ValueError(f"[micro_engram] {what} of {value} is out of range")
    return value


def _check_temperature(value):
    return _check_number(value, "temperature", 1e-6, 1e6)


def _choice(table, value, what):
    try:
        return table[value]
    except KeyError:
        raise ValueError(f"[micro_engram] unknown {what} {value!r}: one of {', '.join(table)}") from None


def _per_row(values, shape, what):
    """fp32 contiguous values of the rows, without their history."""
    if values.shape != shape:
        raise ValueError(f"[micro_engram] {what} {tuple(values.shape)} do not match the rows {tuple(shape)}")
    if values.dtype is torch.float32 and not values.requires_grad and values.is_contiguous():
        return values
    if not values.is_floating_point():
        raise TypeError(f"[micro_engram] {what} must be floating point, got {values.dtype}")
    return values.detach().float().contiguous()


def _sequences(targets, cu_seqlens):
    """(number of sequences, their length where all have one)."""
    if cu_seqlens is None:
        length = targets.shape[-1] if targets.dim() else 1
        return math.prod(targets.shape[:-1]), length
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError(f"[micro_engram] cu_seqlens must be [sequences + 1], got {tuple(cu_seqlens.shape)}")
    if cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"[micro_engram] cu_seqlens must be int32 or int64, got {cu_seqlens.dtype}")
    return cu_seqlens.numel() - 1, 0


def _no_second_derivatives(backward):
    """once_differentiable, whose bookkeeping is needed only where a graph of the backward is made."""
    guarded = once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        return (guarded if torch.is_grad_enabled() else backward)(ctx, *grads)
    return run


def _upstream(grad):
    """The loss's own gradient as the kernels read it."""
    return grad if grad.dtype is torch.float32 and grad.is_contiguous() else grad.float().contiguous()


def _wants_grad(logits):
    return torch.is_grad_enabled() and logits.requires_grad


# ------------------------------------------------------------------------- log-probabilities
# The Functions take everything but their first two tensors as one tuple: apply() costs host time for each argument,
# and a small batch's training step is bound by the rate at which the host issues it. For plain tensors the
# backward's call is made ready in the forward (ctx.run, used once: a second backward makes its own). It holds the
# logits and for two of the losses the gradient, so it is not made where hooks on saved tensors are to have these.
def _makes_ready(*tensors):
    """tensors: all that the call takes, those that were not given as None."""
    return loss_ops.is_plain(*tensors) and torch._C._autograd._top_saved_tensors_default_hooks(False) is None


class _TokenLogps(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, args):
        ctx.run = None
        if _makes_ready(logits, targets):
            (logps, stats), held = loss_ops.run_token_logps(logits.detach(), targets, *args, True)
            ctx.run = loss_ops.LogpsBackward(held, args[1], stats)
        else:
            logps, stats = loss_ops.token_logps(logits.detach(), targets, *args, True)
        ctx.save_for_backward(logits, targets, stats)
        ctx.consts = args
        return logps

    @staticmethod
    @_no_second_derivatives
    def backward(ctx, grad):
        logits, targets, stats = ctx.saved_tensors  # looks whether they are still as they were
        run, ctx.run = ctx.run, None  # so that a loss that is kept does not keep the logits
        if run is not None and type(grad) is torch.Tensor:  # subclasses go through the op
            return run(_upstream(grad)), None, None
        grad = loss_ops.token_logps_backward(logits.detach(), targets, stats, _upstream(grad), *ctx.consts)
        return grad, None, None


def token_logps(logits, targets, temperature=1.0, ignore_index=IGNORE_INDEX):
    """log softmax(logits / temperature) at `targets`: fp32 of targets' shape, 0 where a row does not
    count. Differentiable in the logits."""
    _check_targets(logits, targets)
    temperature, ignore_index = _check_temperature(temperature), int(ignore_index)
    if _wants_grad(logits):
        return _TokenLogps.apply(logits, targets, (ignore_index, temperature))
    return loss_ops.token_logps(logits.detach(), targets, ignore_index, temperature, False)[0]


# -------------------------------------------------------------------------------- preference
class _Preference(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, args):
        ctx.run = None
        if _makes_ready(logits, targets, *args[:2]):  # ref_logps, cu_seqlens
            (loss, chosen, rejected, saved), held = loss_ops.run_preference(logits.detach(), targets, *args, True)
            ctx.run = loss_ops.token_backward(held, 1.0, saved)
        else:
            loss, chosen, rejected, saved = loss_ops.preference(logits.detach(), targets, *args, True)
        ctx.save_for_backward(logits, targets, saved)
        ctx.ignore_index = args[-1]
        ctx.mark_non_differentiable(chosen, rejected)
        ctx.set_materialize_grads(False)
        return loss, chosen, rejected

    @staticmethod
    @_no_second_derivatives
    def backward(ctx, upstream, _chosen, _rejected):
        if upstream is None:
            return None, None, None
        logits, targets, saved = ctx.saved_tensors
        run, ctx.run = ctx.run, None
        if run is not None and type(upstream) is torch.Tensor:
            return run(_upstream(upstream)), None, None
        grad = loss_ops.saved_token_backward(logits.detach(), targets, saved, _upstream(upstream), ctx.ignore_index, 1.0)
        return grad, None, None


def preference_loss(logits, targets, ref_logps, cu_seqlens=None, beta=0.1, loss_type="sigmoid",
                    label_smoothing=0.0, length_normalized=False, ignore_index=IGNORE_INDEX):
    """(loss, chosen rewards [pairs], rejected rewards [pairs]) of preference pairs: the mean over pairs
    of a loss of h = D(chosen) - D(rejected), D of a sequence the sum over its counted tokens of
    (log-probability - ref_logps), or their mean with length_normalized; the rewards are beta D and
    carry no gradient.

    Sequences are the rows of `targets`' last dim, or with cu_seqlens [sequences + 1] (ascending) the rows packed
    back to back; the first half of them are the chosen answers, the second half the rejected ones in the same
    order. ref_logps: the reference's log-probabilities of the same targets (token_logps), token by token:
    differences of single tokens lose nothing, where those of whole sequences' sums would.

    loss_type "sigmoid": -(1 - s) log sigmoid(beta h) - s log sigmoid(-beta h), s the label_smoothing;
    "ipo": (h - 1 / (2 beta))^2; "hinge": max(0, 1 - beta h). A sequence without a counted token has
    D = 0; no pairs at all give 0."""
    _check_targets(logits, targets)
    kind = _choice(_PAIR_LOSSES, loss_type, "loss_type")
    beta = _check_number(beta, "beta", 0.0, 1e6, open_low=True)
    smoothing = _check_number(label_smoothing, "label_smoothing", 0.0, 1.0)
    if smoothing and loss_type != "sigmoid":
        raise ValueError("[micro_engram] label_smoothing is for the sigmoid loss")
    if cu_seqlens is None and targets.dim() < 2:
        raise ValueError("[micro_engram] packed rows need cu_seqlens")
    n_seqs, seq_len = _sequences(targets, cu_seqlens)
    if n_seqs % 2:
        raise ValueError(f"[micro_engram] {n_seqs} sequences are no pairs")
    ref = _per_row(ref_logps, targets.shape, "ref_logps")
    args = (ref, cu_seqlens, n_seqs // 2, seq_len, kind, beta, smoothing, bool(length_normalized), int(ignore_index))
    if _wants_grad(logits):
        return _Preference.apply(logits, targets, args)
    return tuple(loss_ops.preference(logits.detach(), targets, *args, False))


# ------------------------------------------------------------------------------------ policy
class _Policy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, args):
        ctx.consts = args[-1], args[-4]  # ignore_index, temperature
        ctx.run = None
        if _makes_ready(logits, targets, *args[:2], *args[3:5]):  # old_logps, advantages, ref_logps, cu_seqlens
            (loss, logps, out_stats, saved, grad), held = loss_ops.run_policy(logits.detach(), targets, *args, True)
            ctx.run = loss_ops.token_backward(held, args[-4], saved, grad)
        else:  # the gradient is the backward's, nothing is written in place
            loss, logps, out_stats, saved = loss_ops.policy(logits.detach(), targets, *args, False)
        ctx.save_for_backward(logits, targets, saved)
        ctx.mark_non_differentiable(logps, out_stats)
        ctx.set_materialize_grads(False)
        return loss, logps, out_stats

    @staticmethod
    @_no_second_derivatives
    def backward(ctx, upstream, _logps, _stats):
        if upstream is None:
            return None, None, None
        logits, targets, saved = ctx.saved_tensors
        run, ctx.run = ctx.run, None  # its gradient is handed out once
        if run is not None and type(upstream) is torch.Tensor:
            return run(_upstream(upstream)), None, None
        grad = loss_ops.saved_token_backward(logits.detach(), targets, saved, _upstream(upstream), *ctx.consts)
        return grad, None, None


def policy_loss(logits, targets, old_logps, advantages, ref_logps=None, cu_seqlens=None, clip_low=0.2,
                clip_high=0.2, kl_coef=0.0, temperature=1.0, scale=1.0, reduction="token",
                ignore_index=IGNORE_INDEX):
    """(loss, log-probabilities, stats) of sampled tokens: per counted token, with r = exp(logp - old_logps)
    and d = ref_logps - logp,

        -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(d) - d - 1)

    times `scale`, reduced by "token" (mean over counted tokens), "sequence" (mean over sequences with a
    counted token of their means) or "sum". Log-probabilities (fp32, targets' shape) and stats carry no
    gradient; stats [2] are the means over counted tokens of exp(d) - d - 1 (0 without ref_logps; with a kl_coef
    of 0 ref_logps is for this alone) and of the tokens whose ratio was clipped.

    advantages: of targets' shape, or one for each sequence: [sequences], or [sequences, 1], which is never taken
    for values of the tokens where a packed 1-D batch has as many sequences (some of them empty) as tokens, or
    [*targets.shape[:-1], 1] where these are as many. Sequences as in preference_loss (a 1-D batch without
    cu_seqlens is one sequence)."""
    _check_targets(logits, targets)
    how = _choice(_POLICY_REDUCTIONS, reduction, "reduction")
    clip_low = _check_number(clip_low, "clip_low")
    clip_high = _check_number(clip_high, "clip_high")
    kl_coef = _check_number(kl_coef, "kl_coef", -1e6, 1e6)
    scale = _check_number(scale, "scale", -1e30, 1e30)
    temperature = _check_temperature(temperature)
    if kl_coef and ref_logps is None:
        raise ValueError("[micro_engram] kl_coef needs ref_logps")
    n_seqs, seq_len = _sequences(targets, cu_seqlens)
    old = _per_row(old_logps, targets.shape, "old_logps")
    ref = None if ref_logps is None else _per_row(ref_logps, targets.shape, "ref_logps")
    per_seq = advantages.shape != targets.shape
    # one for each of targets.shape[:-1] only where these are all sequences: cu_seqlens may name more than they hold
    if per_seq and (advantages.numel() != n_seqs or tuple(advantages.shape) not in
                    ((n_seqs,), (n_seqs, 1), (*targets.shape[:-1], 1))):
        raise ValueError(f"[micro_engram] advantages {tuple(advantages.shape)} are neither the rows' "
                         f"{tuple(targets.shape)} nor one for each of {n_seqs} sequences")
    adv = _per_row(advantages, advantages.shape, "advantages")
    args = (old, adv, per_seq, ref, cu_seqlens, n_seqs, seq_len, clip_low, clip_high, kl_coef, temperature, scale,
            how, int(ignore_index))
    if _wants_grad(logits):
        return _Policy.apply(logits, targets, args)
    return tuple(loss_ops.policy(logits.detach(), targets, *args, False)[:3])


# ------------------------------------------------------------------------------ distillation
class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_ids, args):
        ctx.temperature = args[3]
        ctx.run = None
        if _makes_ready(logits, teacher_ids, *args[:3]):  # teacher_logits, teacher_lse, mask
            (loss, saved, grad), held = loss_ops.run_distill(logits.detach(), teacher_ids, *args, True)
            ctx.run = loss_ops.distill_backward_of(held, ctx.temperature, saved, grad)
        else:
            loss, saved = loss_ops.distill(logits.detach(), teacher_ids, *args, False)
        ctx.save_for_backward(logits, teacher_ids, saved)
        return loss

    @staticmethod
    @_no_second_derivatives
    def backward(ctx, upstream):
        logits, teacher_ids, saved = ctx.saved_tensors
        run, ctx.run = ctx.run, None
        if run is not None and type(upstream) is torch.Tensor:
            return run(_upstream(upstream)), None, None
        grad = loss_ops.distill_backward(logits.detach(), teacher_ids, saved, _upstream(upstream), ctx.temperature)
        return grad, None, None


def distill_loss(logits, teacher_ids, teacher_logits, teacher_lse=None, mask=None, temperature=1.0, scale=1.0,
                 reduction="mean"):
    """temperature^2 KL(teacher | softmax(logits / temperature)) times `scale`, the mean (or "sum") over the
    rows that count, from the teacher's top entries of each row.

    teacher_ids [..., top] (int32 / int64) and teacher_logits [..., top] (bf16 / fp32): token and logit of
    each entry, up to 1024 of them in any order. Entries whose id is no token (-1) are left out, and a row of only
    such does not count; entries of one token add up.
    teacher_lse: None takes the teacher's softmax over the entries alone. Else fp32 [...], the log of the
    sum over its whole vocabulary of exp(teacher logit / temperature): an entry's probability is then
    its real one, and all tokens that are no entry are one class more with what is left (stored
    log-probabilities at temperature 1 come with teacher_lse = 0).
    mask [...] (bool): rows that count, None for all."""
    _check_logits(logits)
    lead = tuple(logits.shape[:-1])
    if teacher_ids.dim() != logits.dim() or tuple(teacher_ids.shape[:-1]) != lead:
        raise ValueError(f"[micro_engram] teacher_ids {tuple(teacher_ids.shape)} do not match the logits' rows {lead}")
    if tuple(teacher_logits.shape) != tuple(teacher_ids.shape):
        raise ValueError(f"[micro_engram] teacher_logits {tuple(teacher_logits.shape)} do not match teacher_ids "
                         f"{tuple(teacher_ids.shape)}")
    if teacher_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"[micro_engram] teacher_ids must be int32 or int64, got {teacher_ids.dtype}")
    if teacher_logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"[micro_engram] teacher_logits must be bf16 or fp32, got {teacher_logits.dtype}")
    if not 1 <= teacher_ids.shape[-1] <= TOP_MAX:
        raise ValueError(f"[micro_engram] {teacher_ids.shape[-1]} teacher entries: 1 to {TOP_MAX} are taken")
    temperature, scale = _check_temperature(temperature), _check_number(scale, "scale", -1e30, 1e30)
    how = _choice(_DISTILL_REDUCTIONS, reduction, "reduction")
    lse = None
    if teacher_lse is not None:
        lse = _per_row(teacher_lse, lead, "teacher_lse")
        if teacher_ids.shape[-1] >= logits.shape[-1]:
            raise ValueError("[micro_engram] teacher entries for every token leave no rest for teacher_lse")
    if mask is not None:
        if tuple(mask.shape) != lead or mask.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"[micro_engram] mask must be bool {lead}, got {mask.dtype} {tuple(mask.shape)}")
        mask = mask.contiguous()
    args = (teacher_logits.detach(), lse, mask, temperature, scale, how)
    if _wants_grad(logits):
        return _Distill.apply(logits, teacher_ids, args)
    return loss_ops.distill(logits.detach(), teacher_ids, *args, False)[0]
