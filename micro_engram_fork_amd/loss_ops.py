"""torch custom ops over the loss entry points of libmicro_engram_amd.so (csrc/losses.hip), in the
manner of ops.py: outputs and workspaces from torch's allocator, kernels on the current stream, a
fake implementation for tracing, no host synchronisation. losses.py is the surface for users.
"""
import ctypes
import functools
import math
from typing import List, Optional

import torch

from ._lib import ME_I32, ME_I64, call
from .ops import _custom_op, _direct_call, _p, dtype_code, require_gpu, stream_of


@functools.lru_cache(maxsize=256)
def workspace_bytes(n, vocab, pairs=0, top=0):
    size = ctypes.c_size_t(0)
    call("me_loss_workspace_size", n, vocab, pairs, top, ctypes.byref(size))
    return size.value


def _workspace(n, vocab, dev, pairs=0, top=0):
    ws = torch.empty(workspace_bytes(n, vocab, pairs, top), dtype=torch.uint8, device=dev)
    return ws, ws.data_ptr(), ws.numel()


def row_layout(logits):
    """(logits, the C-ABI's seven arguments of them): rows of a strided tensor as they lie, whether a
    view of a longer sequence or of a padded vocabulary; copied only where the values of a row are
    not next to each other, or the leading dims are not two strides."""
    vocab = logits.shape[-1]
    if logits.stride(-1) != 1 and vocab > 1:
        logits = logits.contiguous()
    lead = logits.dim() - 1
    n = logits.numel() // vocab if vocab else 0
    rows = logits
    if lead > 2:
        flat = math.prod(logits.shape[:-2]), logits.shape[-2], vocab
        try:
            rows = logits.view(flat)
        except RuntimeError:
            logits = logits.contiguous()
            rows = logits.view(flat)
    if lead == 0:
        per, batch_stride, row_stride = 1, 0, 0
    elif lead == 1:
        per, batch_stride, row_stride = max(1, n), 0, rows.stride(0)
    else:
        per, batch_stride, row_stride = max(1, rows.shape[1]), rows.stride(0), rows.stride(1)
    return logits, (logits.data_ptr(), dtype_code(logits), n, vocab, per, batch_stride, row_stride)


def is_plain(*tensors):
    """Whether a call on these tensors runs the kernels at once (no tracing, no fake tensors)."""
    return _direct_call(tensors, None)


def _int_code(t, what):
    if t.dtype is torch.int64:
        return ME_I64
    if t.dtype is torch.int32:
        return ME_I32
    raise TypeError(f"[micro_engram] {what} must be int32 or int64, got {t.dtype}")


def _contiguous(t):
    return t if t.is_contiguous() else t.contiguous()


def _targets(targets, ignore_index):
    targets = _contiguous(targets)
    return targets, (targets.data_ptr(), _int_code(targets, "targets"), ignore_index)


def _offsets(offsets):
    if offsets is None:
        return None, (None, 0)
    offsets = _contiguous(offsets)
    return offsets, (offsets.data_ptr(), _int_code(offsets, "cu_seqlens"))


def _f32(shape, dev):
    return torch.empty(shape, dtype=torch.float32, device=dev)


# What a backward needs of n rows is one fp32 buffer: statistics [n, 4], factors [n], and for
# distillation the values at the teacher's entries [n, top].
def _saved(n, dev, top=0):
    """(buffer, addresses of its parts)."""
    saved = _f32(n * (5 + top), dev)
    return saved, *_saved_parts(saved, n)


def _saved_parts(saved, n):
    at = saved.data_ptr()
    return at, at + 16 * n, at + 20 * n


# ------------------------------------------------------------------------- log-probabilities
def run_token_logps(logits, targets, ignore_index, temperature, with_stats):
    """([log-probabilities, stats or None], arguments of the rows and tokens with the tensors that hold them)."""
    dev = require_gpu(logits, targets)
    logits, rows = row_layout(logits)
    targets, toks = _targets(targets, ignore_index)
    n, vocab = rows[2], rows[3]
    out = _f32(targets.shape, dev)
    stats = _f32((n, 4), dev) if with_stats else None
    ws, ptr, size = _workspace(n, vocab, dev)
    call("me_token_logps", *rows, *toks, temperature, out.data_ptr(), _p(stats), ptr, size, stream_of(dev))
    return [out, stats], ((*rows, *toks), logits, targets)


@_custom_op("token_logps")
def token_logps(logits: torch.Tensor, targets: torch.Tensor, ignore_index: int, temperature: float,
                with_stats: bool) -> List[torch.Tensor]:
    """[log-probabilities fp32 of targets' shape], plus row stats [n, 4] (what the backward needs)
    when with_stats."""
    res, _ = run_token_logps(logits, targets, ignore_index, temperature, with_stats)
    return res if with_stats else res[:1]


@token_logps.register_fake
def _(logits, targets, ignore_index, temperature, with_stats):
    out = logits.new_empty(targets.shape, dtype=torch.float32)
    return [out, logits.new_empty((targets.numel(), 4), dtype=torch.float32)] if with_stats else [out]


def _token_logps_backward(logits, targets, stats, coef, upstream, ignore_index, temperature, coef_scale):
    """stats, coef: addresses."""
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    logits, rows = row_layout(logits)
    targets, toks = _targets(targets, ignore_index)
    call("me_token_logps_backward", *rows, *toks, temperature, stats, coef, coef_scale, _p(upstream),
         0, grad.data_ptr(), stream_of(logits.device))
    return grad


@_custom_op("token_logps_backward")
def token_logps_backward(logits: torch.Tensor, targets: torch.Tensor, stats: torch.Tensor, coef: torch.Tensor,
                         ignore_index: int, temperature: float) -> torch.Tensor:
    """The logits' gradient coef / temperature * (1[j = target] - probability of j)."""
    require_gpu(logits, targets, stats, coef)
    return _token_logps_backward(logits, targets, stats.data_ptr(), coef.data_ptr(), None, ignore_index, temperature,
                                 1.0 / temperature)


@token_logps_backward.register_fake
def _(logits, targets, stats, coef, ignore_index, temperature):
    return logits.new_empty(logits.shape)


@_custom_op("saved_token_backward")
def saved_token_backward(logits: torch.Tensor, targets: torch.Tensor, saved: torch.Tensor, upstream: torch.Tensor,
                         ignore_index: int, temperature: float) -> torch.Tensor:
    """The logits' gradient from what preference and policy leave of their rows, times upstream (fp32)."""
    require_gpu(logits, targets, saved, upstream)
    stats, coef, _ = _saved_parts(saved, targets.numel())
    return _token_logps_backward(logits, targets, stats, coef, upstream, ignore_index, temperature, 1.0)


@saved_token_backward.register_fake
def _(logits, targets, saved, upstream, ignore_index, temperature):
    return logits.new_empty(logits.shape)


# A backward's call, made ready in the forward, which has the arguments at hand: autograd runs the backward in a thread
# of its own, where everything takes longer. Not for traced calls.
class Backward:
    """backward(upstream): the logits' gradient by the entry point `name` with `args` up to its upstream argument.
    grad: the gradient for an upstream of 1, which the forward has written already; it is made the one for
    `upstream` in place, and only where that is not 1 (the kernel looks, not the host). None: a new one.
    kept: tensors behind the addresses in args."""
    __slots__ = ("name", "args", "like", "grad", "kept")

    def __init__(self, name, args, like, grad, kept):
        self.name, self.args, self.like, self.grad, self.kept = name, args, like, grad, kept

    def __call__(self, upstream):
        grad, done = self.grad, 1
        if grad is None:
            grad, done = torch.empty(self.like.shape, dtype=self.like.dtype, device=self.like.device), 0
        call(self.name, *self.args, upstream.data_ptr(), done, grad.data_ptr(), stream_of(grad.device))
        return grad


class LogpsBackward:
    """As Backward, for token_logps, whose upstream is a factor for each row."""
    __slots__ = ("args", "scale", "like", "kept")

    def __init__(self, held, temperature, stats):
        args, self.like, targets = held
        self.args, self.scale, self.kept = (*args, temperature, stats.data_ptr()), 1.0 / temperature, (targets, stats)

    def __call__(self, upstream):
        grad = torch.empty(self.like.shape, dtype=self.like.dtype, device=self.like.device)
        call("me_token_logps_backward", *self.args, upstream.data_ptr(), self.scale, None, 0, grad.data_ptr(),
             stream_of(grad.device))
        return grad


def token_backward(held, temperature, saved, grad=None):
    """Backward of preference and policy. held: as run_policy gives it."""
    args, logits, targets = held
    stats, coef, _ = _saved_parts(saved, args[2])
    return Backward("me_token_logps_backward", (*args, temperature, stats, coef, 1.0), logits, grad, (targets, saved))


def distill_backward_of(held, temperature, saved, grad):
    args, logits, ids = held
    return Backward("me_distill_backward", (*args, temperature, *_saved_parts(saved, args[2])), logits, grad,
                    (ids, saved))


# -------------------------------------------------------------------------------- preference
def run_preference(logits, targets, ref_logps, offsets, pairs, seq_len, kind, beta, smoothing, normalized,
                   ignore_index, with_saved):
    """([loss, chosen, rejected, saved or None], held as of run_token_logps)."""
    dev = require_gpu(logits, targets, ref_logps, offsets)
    logits, rows = row_layout(logits)
    targets, toks = _targets(targets, ignore_index)
    offsets, seqs = _offsets(offsets)
    n, vocab = rows[2], rows[3]
    loss, chosen, rejected = _f32((), dev), _f32((pairs,), dev), _f32((pairs,), dev)
    saved, stats, coef, _ = _saved(n, dev) if with_saved else (None,) * 4
    ws, ptr, size = _workspace(n, vocab, dev, pairs)
    call("me_preference", *rows, *toks, ref_logps.data_ptr(), *seqs, pairs, seq_len, kind, beta, smoothing,
         int(normalized), loss.data_ptr(), chosen.data_ptr(), rejected.data_ptr(), stats, coef, ptr, size,
         stream_of(dev))
    return [loss, chosen, rejected, saved], ((*rows, *toks), logits, targets)


@_custom_op("preference")
def preference(logits: torch.Tensor, targets: torch.Tensor, ref_logps: torch.Tensor,
               offsets: Optional[torch.Tensor], pairs: int, seq_len: int, kind: int, beta: float,
               smoothing: float, normalized: bool, ignore_index: int, with_saved: bool) -> List[torch.Tensor]:
    """[loss, chosen [pairs], rejected [pairs]], plus saved [5 n] (what the backward needs) when
    with_saved, all fp32."""
    res, _ = run_preference(logits, targets, ref_logps, offsets, pairs, seq_len, kind, beta, smoothing, normalized,
                            ignore_index, with_saved)
    return res if with_saved else res[:3]


@preference.register_fake
def _(logits, targets, ref_logps, offsets, pairs, seq_len, kind, beta, smoothing, normalized, ignore_index,
      with_saved):
    n, new = targets.numel(), functools.partial(logits.new_empty, dtype=torch.float32)
    res = [new(()), new((pairs,)), new((pairs,))]
    return [*res, new((5 * n,))] if with_saved else res


# ------------------------------------------------------------------------------------ policy
def run_policy(logits, targets, old_logps, advantages, adv_per_seq, ref_logps, offsets, n_seqs, seq_len, clip_low,
               clip_high, kl_coef, temperature, scale, reduction, ignore_index, with_grad):
    """([loss, log-probabilities, stats, saved, gradient or None], held as of run_token_logps)."""
    dev = require_gpu(logits, targets, old_logps, advantages, ref_logps, offsets)
    logits, rows = row_layout(logits)
    targets, toks = _targets(targets, ignore_index)
    offsets, seqs = _offsets(offsets)
    n, vocab = rows[2], rows[3]
    loss, logps, out_stats = _f32((), dev), _f32(targets.shape, dev), _f32((2,), dev)
    saved, stats, coef, _ = _saved(n, dev)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if with_grad else None
    ws, ptr, size = _workspace(n, vocab, dev)
    call("me_policy", *rows, *toks, old_logps.data_ptr(), advantages.data_ptr(), int(adv_per_seq), _p(ref_logps),
         *seqs, n_seqs, seq_len, clip_low, clip_high, kl_coef, temperature, scale, reduction, loss.data_ptr(),
         logps.data_ptr(), out_stats.data_ptr(), stats, coef, _p(grad), ptr, size, stream_of(dev))
    return [loss, logps, out_stats, saved, grad], ((*rows, *toks), logits, targets)


@_custom_op("policy")
def policy(logits: torch.Tensor, targets: torch.Tensor, old_logps: torch.Tensor, advantages: torch.Tensor,
           adv_per_seq: bool, ref_logps: Optional[torch.Tensor], offsets: Optional[torch.Tensor], n_seqs: int,
           seq_len: int, clip_low: float, clip_high: float, kl_coef: float, temperature: float, scale: float,
           reduction: int, ignore_index: int, with_grad: bool) -> List[torch.Tensor]:
    """[loss, log-probabilities of targets' shape, (mean KL, clipped share), saved [5 n]], all fp32, plus
    the logits' gradient for an upstream of 1 when with_grad."""
    res, _ = run_policy(logits, targets, old_logps, advantages, adv_per_seq, ref_logps, offsets, n_seqs, seq_len,
                        clip_low, clip_high, kl_coef, temperature, scale, reduction, ignore_index, with_grad)
    return res if with_grad else res[:4]


@policy.register_fake
def _(logits, targets, old_logps, advantages, adv_per_seq, ref_logps, offsets, n_seqs, seq_len, clip_low,
      clip_high, kl_coef, temperature, scale, reduction, ignore_index, with_grad):
    n, new = targets.numel(), functools.partial(logits.new_empty, dtype=torch.float32)
    res = [new(()), new(targets.shape), new((2,)), new((5 * n,))]
    return [*res, logits.new_empty(logits.shape)] if with_grad else res


# ------------------------------------------------------------------------------ distillation
def run_distill(logits, teacher_ids, teacher_logits, teacher_lse, mask, temperature, scale, reduction, with_grad):
    """([loss, saved, gradient or None], held: the arguments of the rows and ids with their tensors)."""
    dev = require_gpu(logits, teacher_ids, teacher_logits, teacher_lse, mask)
    logits, rows = row_layout(logits)
    n, vocab = rows[2], rows[3]
    ids, teacher = _contiguous(teacher_ids), _contiguous(teacher_logits)
    top = ids.shape[-1]
    loss = _f32((), dev)
    saved, stats, coef, fix = _saved(n, dev, top)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if with_grad else None
    ws, ptr, size = _workspace(n, vocab, dev, 0, top)
    id_args = ids.data_ptr(), _int_code(ids, "teacher_ids")
    call("me_distill", *rows, *id_args, teacher.data_ptr(), dtype_code(teacher), top, _p(teacher_lse), _p(mask),
         temperature, scale, reduction, loss.data_ptr(), stats, coef, fix, _p(grad), ptr, size, stream_of(dev))
    return [loss, saved, grad], ((*rows, *id_args, top), logits, ids)


@_custom_op("distill")
def distill(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
            teacher_lse: Optional[torch.Tensor], mask: Optional[torch.Tensor], temperature: float, scale: float,
            reduction: int, with_grad: bool) -> List[torch.Tensor]:
    """[loss, saved [(5 + top) n]], fp32, plus the logits' gradient for an upstream of 1 when with_grad."""
    res, _ = run_distill(logits, teacher_ids, teacher_logits, teacher_lse, mask, temperature, scale, reduction,
                         with_grad)
    return res if with_grad else res[:2]


@distill.register_fake
def _(logits, teacher_ids, teacher_logits, teacher_lse, mask, temperature, scale, reduction, with_grad):
    top = teacher_ids.shape[-1]
    n, new = teacher_ids.numel() // top, functools.partial(logits.new_empty, dtype=torch.float32)
    res = [new(()), new((n * (5 + top),))]
    return [*res, logits.new_empty(logits.shape)] if with_grad else res


@_custom_op("distill_backward")
def distill_backward(logits: torch.Tensor, teacher_ids: torch.Tensor, saved: torch.Tensor, upstream: torch.Tensor,
                     temperature: float) -> torch.Tensor:
    """The logits' gradient from what distill leaves of its rows, times upstream (fp32)."""
    require_gpu(logits, teacher_ids, saved, upstream)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    logits, rows = row_layout(logits)
    ids = _contiguous(teacher_ids)
    call("me_distill_backward", *rows, ids.data_ptr(), _int_code(ids, "teacher_ids"), ids.shape[-1], temperature,
         *_saved_parts(saved, rows[2]), upstream.data_ptr(), 0, grad.data_ptr(), stream_of(logits.device))
    return grad


@distill_backward.register_fake
def _(logits, teacher_ids, saved, upstream, temperature):
    return logits.new_empty(logits.shape)
