"""torch custom ops over the loss entry points of libmicro_engram_amd.so (csrc/losses.hip), in the
manner of ops.py: outputs and workspaces from torch's allocator, kernels on the current stream, a
fake implementation for tracing, no host synchronisation. losses.py is the surface for users.
"""
import ctypes
import functools
from typing import List, Optional

import torch

from ._lib import ME_I32, ME_I64, call
from .ops import _custom_op, _p, dtype_code, require_gpu, stream_of


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
    if lead > 2:
        try:
            rows = logits.view(-1, logits.shape[-2], vocab)
        except RuntimeError:
            logits = logits.contiguous()
            rows = logits.view(-1, logits.shape[-2], vocab)
    else:
        rows = logits
    if lead == 0:
        per, batch_stride, row_stride = 1, 0, 0
    elif lead == 1:
        per, batch_stride, row_stride = max(1, n), 0, rows.stride(0)
    else:
        per, batch_stride, row_stride = max(1, rows.shape[1]), rows.stride(0), rows.stride(1)
    return logits, (logits.data_ptr(), dtype_code(logits), n, vocab, per, batch_stride, row_stride)


def _int_code(t, what):
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"[micro_engram] {what} must be int32 or int64, got {t.dtype}")
    return ME_I32 if t.dtype == torch.int32 else ME_I64


def _targets(targets, ignore_index):
    targets = targets.contiguous()
    return targets, (targets.data_ptr(), _int_code(targets, "targets"), ignore_index)


def _offsets(offsets):
    if offsets is None:
        return None, (None, 0)
    offsets = offsets.contiguous()
    return offsets, (offsets.data_ptr(), _int_code(offsets, "cu_seqlens"))


def _f32(*shape, dev):
    return torch.empty(shape, dtype=torch.float32, device=dev)


# ------------------------------------------------------------------------- log-probabilities
@_custom_op("token_logps")
def token_logps(logits: torch.Tensor, targets: torch.Tensor, ignore_index: int, temperature: float,
                with_stats: bool) -> List[torch.Tensor]:
    """[log-probabilities fp32 of targets' shape], plus row stats [n, 2] (what the backward needs)
    when with_stats."""
    dev = require_gpu(logits, targets)
    logits, rows = row_layout(logits)
    targets, toks = _targets(targets, ignore_index)
    n, vocab = rows[2], rows[3]
    out = _f32(*targets.shape, dev=dev)
    stats = _f32(n, 2, dev=dev) if with_stats else None
    ws, ptr, size = _workspace(n, vocab, dev)
    call("me_token_logps", *rows, *toks, temperature, out.data_ptr(), _p(stats), ptr, size, stream_of(dev))
    return [out, stats] if with_stats else [out]


@token_logps.register_fake
def _(logits, targets, ignore_index, temperature, with_stats):
    out = logits.new_empty(targets.shape, dtype=torch.float32)
    return [out, logits.new_empty((targets.numel(), 2), dtype=torch.float32)] if with_stats else [out]


def _token_logps_backward(grad, logits, targets, stats, coef, upstream, ignore_index, temperature, coef_scale,
                          done_for_one):
    dev = require_gpu(logits, targets, stats, coef, upstream)
    logits, rows = row_layout(logits)
    targets, toks = _targets(targets, ignore_index)
    call("me_token_logps_backward", *rows, *toks, temperature, stats.data_ptr(), coef.data_ptr(), coef_scale,
         _p(upstream), int(done_for_one), grad.data_ptr(), stream_of(dev))
    return grad


@_custom_op("token_logps_backward")
def token_logps_backward(logits: torch.Tensor, targets: torch.Tensor, stats: torch.Tensor, coef: torch.Tensor,
                         upstream: Optional[torch.Tensor], ignore_index: int, temperature: float,
                         coef_scale: float) -> torch.Tensor:
    """The logits' gradient coef * coef_scale * upstream * (1[j = target] - probability of j)."""
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    return _token_logps_backward(grad, logits, targets, stats, coef, upstream, ignore_index, temperature,
                                 coef_scale, False)


@token_logps_backward.register_fake
def _(logits, targets, stats, coef, upstream, ignore_index, temperature, coef_scale):
    return logits.new_empty(logits.shape)


def token_grad_for(grad, upstream, logits, targets, stats, coef, ignore_index, temperature):
    """`grad`, the gradient for an upstream of 1, made the one for `upstream`: in place, and only where
    that is not 1 (the kernel looks, not the host)."""
    return _token_logps_backward(grad, logits, targets, stats, coef, upstream, ignore_index, temperature, 1.0, True)


# -------------------------------------------------------------------------------- preference
@_custom_op("preference")
def preference(logits: torch.Tensor, targets: torch.Tensor, ref_logps: torch.Tensor,
               offsets: Optional[torch.Tensor], pairs: int, seq_len: int, kind: int, beta: float,
               smoothing: float, normalized: bool, ignore_index: int) -> List[torch.Tensor]:
    """[loss, chosen [pairs], rejected [pairs], row stats [n, 2], coef [n]], all fp32."""
    dev = require_gpu(logits, targets, ref_logps, offsets)
    logits, rows = row_layout(logits)
    targets, toks = _targets(targets, ignore_index)
    offsets, seqs = _offsets(offsets)
    n, vocab = rows[2], rows[3]
    loss, chosen, rejected = _f32(dev=dev), _f32(pairs, dev=dev), _f32(pairs, dev=dev)
    stats, coef = _f32(n, 2, dev=dev), _f32(n, dev=dev)
    ws, ptr, size = _workspace(n, vocab, dev, pairs)
    call("me_preference", *rows, *toks, ref_logps.data_ptr(), *seqs, pairs, seq_len, kind, beta, smoothing,
         int(normalized), loss.data_ptr(), chosen.data_ptr(), rejected.data_ptr(), stats.data_ptr(),
         coef.data_ptr(), ptr, size, stream_of(dev))
    return [loss, chosen, rejected, stats, coef]


@preference.register_fake
def _(logits, targets, ref_logps, offsets, pairs, seq_len, kind, beta, smoothing, normalized, ignore_index):
    n, new = targets.numel(), functools.partial(logits.new_empty, dtype=torch.float32)
    return [new(()), new((pairs,)), new((pairs,)), new((n, 2)), new((n,))]


# ------------------------------------------------------------------------------------ policy
@_custom_op("policy")
def policy(logits: torch.Tensor, targets: torch.Tensor, old_logps: torch.Tensor, advantages: torch.Tensor,
           adv_per_seq: bool, ref_logps: Optional[torch.Tensor], offsets: Optional[torch.Tensor], n_seqs: int,
           seq_len: int, clip_low: float, clip_high: float, kl_coef: float, temperature: float, scale: float,
           reduction: int, ignore_index: int, with_grad: bool) -> List[torch.Tensor]:
    """[loss, log-probabilities of targets' shape, (mean KL, clipped share), row stats [n, 2], coef [n]],
    all fp32, plus the logits' gradient for an upstream of 1 when with_grad."""
    dev = require_gpu(logits, targets, old_logps, advantages, ref_logps, offsets)
    logits, rows = row_layout(logits)
    targets, toks = _targets(targets, ignore_index)
    offsets, seqs = _offsets(offsets)
    n, vocab = rows[2], rows[3]
    loss, logps, out_stats = _f32(dev=dev), _f32(*targets.shape, dev=dev), _f32(2, dev=dev)
    stats, coef = _f32(n, 2, dev=dev), _f32(n, dev=dev)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if with_grad else None
    ws, ptr, size = _workspace(n, vocab, dev)
    call("me_policy", *rows, *toks, old_logps.data_ptr(), advantages.data_ptr(), int(adv_per_seq), _p(ref_logps),
         *seqs, n_seqs, seq_len, clip_low, clip_high, kl_coef, temperature, scale, reduction, loss.data_ptr(),
         logps.data_ptr(), out_stats.data_ptr(), stats.data_ptr(), coef.data_ptr(), _p(grad), ptr, size,
         stream_of(dev))
    res = [loss, logps, out_stats, stats, coef]
    return [*res, grad] if with_grad else res


@policy.register_fake
def _(logits, targets, old_logps, advantages, adv_per_seq, ref_logps, offsets, n_seqs, seq_len, clip_low,
      clip_high, kl_coef, temperature, scale, reduction, ignore_index, with_grad):
    n, new = targets.numel(), functools.partial(logits.new_empty, dtype=torch.float32)
    res = [new(()), new(targets.shape), new((2,)), new((n, 2)), new((n,))]
    return [*res, logits.new_empty(logits.shape)] if with_grad else res


# ------------------------------------------------------------------------------ distillation
@_custom_op("distill")
def distill(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
            teacher_lse: Optional[torch.Tensor], mask: Optional[torch.Tensor], temperature: float, scale: float,
            reduction: int, with_grad: bool) -> List[torch.Tensor]:
    """[loss, row stats [n, 2], coef [n], fix [n, top]], all fp32, plus the logits' gradient for an
    upstream of 1 when with_grad."""
    dev = require_gpu(logits, teacher_ids, teacher_logits, teacher_lse, mask)
    logits, rows = row_layout(logits)
    n, vocab = rows[2], rows[3]
    ids, teacher = teacher_ids.contiguous(), teacher_logits.contiguous()
    top = ids.shape[-1]
    loss, stats, coef, fix = _f32(dev=dev), _f32(n, 2, dev=dev), _f32(n, dev=dev), _f32(n, top, dev=dev)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if with_grad else None
    ws, ptr, size = _workspace(n, vocab, dev, 0, top)
    call("me_distill", *rows, ids.data_ptr(), _int_code(ids, "teacher_ids"), teacher.data_ptr(),
         dtype_code(teacher), top, _p(teacher_lse), _p(mask), temperature, scale, reduction, loss.data_ptr(),
         stats.data_ptr(), coef.data_ptr(), fix.data_ptr(), _p(grad), ptr, size, stream_of(dev))
    res = [loss, stats, coef, fix]
    return [*res, grad] if with_grad else res


@distill.register_fake
def _(logits, teacher_ids, teacher_logits, teacher_lse, mask, temperature, scale, reduction, with_grad):
    top = teacher_ids.shape[-1]
    n, new = teacher_ids.numel() // top, functools.partial(logits.new_empty, dtype=torch.float32)
    res = [new(()), new((n, 2)), new((n,)), new((n, top))]
    return [*res, logits.new_empty(logits.shape)] if with_grad else res


def _distill_backward(grad, logits, teacher_ids, stats, coef, fix, upstream, temperature, done_for_one):
    dev = require_gpu(logits, teacher_ids, stats, coef, fix, upstream)
    logits, rows = row_layout(logits)
    ids = teacher_ids.contiguous()
    call("me_distill_backward", *rows, ids.data_ptr(), _int_code(ids, "teacher_ids"), ids.shape[-1], temperature,
         stats.data_ptr(), coef.data_ptr(), fix.data_ptr(), _p(upstream), int(done_for_one), grad.data_ptr(),
         stream_of(dev))
    return grad


@_custom_op("distill_backward")
def distill_backward(logits: torch.Tensor, teacher_ids: torch.Tensor, stats: torch.Tensor, coef: torch.Tensor,
                     fix: torch.Tensor, upstream: Optional[torch.Tensor], temperature: float) -> torch.Tensor:
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    return _distill_backward(grad, logits, teacher_ids, stats, coef, fix, upstream, temperature, False)


@distill_backward.register_fake
def _(logits, teacher_ids, stats, coef, fix, upstream, temperature):
    return logits.new_empty(logits.shape)


def distill_grad_for(grad, upstream, logits, teacher_ids, stats, coef, fix, temperature):
    """As token_grad_for."""
    return _distill_backward(grad, logits, teacher_ids, stats, coef, fix, upstream, temperature, True)
