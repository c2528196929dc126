"""torch custom ops over the head entry points of libmicro_engram_amd.so (csrc/head.hip), in the manner of
loss_ops.py. losses.py is the surface for users.
"""
import ctypes
import functools
from typing import List, Optional

import torch

from ._lib import call
from .loss_ops import _targets, row_layout
from .ops import _custom_op, _p, call_on, dtype_code, require_gpu

_FORWARD, _BACKWARD, _FORWARD_UNIT, _BACKWARD_UNIT = 0, 1, 2, 3
NO_GRADIENT, OF_HIDDEN, OF_WEIGHT = 0, 1, 2  # what a forward may leave something for: hidden alone, weight as well


def weight_layout(weight):
    """(weight, its address, rows and row stride): as it lies where its rows are apart by their length or more."""
    vocab, dim = weight.shape
    if (weight.stride(1) != 1 and dim > 1) or (weight.stride(0) < dim and vocab > 1):
        weight = weight.contiguous()
    return weight, (weight.data_ptr(), vocab, max(weight.stride(0), dim))


def _operands(hidden, weight, targets, ignore_index):
    """(tensors to hold, the entry points' arguments up to the targets')."""
    hidden, rows = row_layout(hidden)
    weight, head = weight_layout(weight)
    targets, toks = _targets(targets, ignore_index)
    return (hidden, weight, targets), (*rows, *head, *toks)


@functools.lru_cache(maxsize=256)
def workspace_bytes(n, vocab, dim, dtype, misaligned, w_stride, which, smoothed):
    """misaligned: the weight's address modulo 16."""
    size = ctypes.c_size_t(0)
    call("me_head_workspace_size", n, vocab, dim, dtype, misaligned, w_stride, which, smoothed, ctypes.byref(size))
    return size.value


def _workspace(operands, dev, which, smoothed=False):
    """(buffer, address, size)."""
    _, dtype, n, dim, _, _, _, weight, vocab, w_stride = operands[:10]
    ws = torch.empty(workspace_bytes(n, vocab, dim, dtype, weight % 16, w_stride, which, smoothed), dtype=torch.uint8, device=dev)
    return ws, ws.data_ptr(), ws.numel()


@functools.lru_cache(maxsize=256)
def unit_elements(n, vocab, dim, dtype, gradients):
    """Size of what a forward leaves for these gradients; 0: nothing."""
    if gradients == NO_GRADIENT:
        return 0
    size = ctypes.c_int64(0)
    call("me_head_unit_size", n, vocab, dim, dtype, int(gradients == OF_WEIGHT), ctypes.byref(size))
    return size.value


def _forward(name, hidden, weight, targets, ignore_index, gradients, out, args):
    """([out, saved] and unit where the call leaves one, the operands' arguments with the tensors that hold them)."""
    dev = require_gpu(hidden, weight, targets)
    held, operands = _operands(hidden, weight, targets, ignore_index)
    saved = torch.empty(16 + 5 * operands[2], dtype=torch.float32, device=dev)
    size = unit_elements(operands[2], operands[8], operands[3], operands[1], gradients)
    unit = torch.empty(size, dtype=torch.float32, device=dev) if size else None
    smoothed = len(args) > 1 and args[1] != 0.0
    ws, ptr, size = _workspace(operands, dev, _FORWARD if unit is None else _FORWARD_UNIT, smoothed)
    call_on(dev, name, *operands, *args, out.data_ptr(), saved.data_ptr(), _p(unit), ptr, size)
    return [out, saved] if unit is None else [out, saved, unit], (held, operands)


class Backward:
    """The backward's call, made ready in the forward: as loss_ops.Backward. kept: what the forward gave beside its result;
    consts: the arguments of head_backward from the temperature to the reduction."""
    __slots__ = ("held", "operands", "saved", "unit", "consts")

    def __init__(self, held, kept, consts):
        (self.held, self.operands), self.consts = held, consts
        self.saved, self.unit = kept[0], kept[1] if len(kept) > 1 else None

    def __call__(self, upstream, need_hidden, need_weight):
        hidden, weight, _ = self.held
        return _backward(hidden.shape, weight.shape, self.operands, hidden, self.saved, self.unit, upstream, self.consts,
                         need_hidden, need_weight)


def _backward(hidden_shape, weight_shape, operands, like, saved, unit, upstream, consts, need_hidden, need_weight):
    """(gradient of hidden or None, gradient of weight or None)."""
    dev, dtype = like.device, like.dtype
    grad_hidden = torch.empty(hidden_shape, dtype=dtype, device=dev) if need_hidden else None
    grad_weight = torch.empty(weight_shape, dtype=dtype, device=dev) if need_weight else None
    ws, ptr, size = _workspace(operands, dev, _BACKWARD if unit is None else _BACKWARD_UNIT)
    temperature, per_row, smoothing, z_loss, scale, reduction = consts
    call_on(dev, "me_head_backward", *operands, temperature, upstream.data_ptr(), int(per_row), smoothing, z_loss, scale,
            reduction, saved.data_ptr(), _p(unit), _p(grad_hidden), _p(grad_weight), ptr, size)
    return grad_hidden, grad_weight


def _fake_forward(hidden, weight, targets, gradients, shape):
    res = [hidden.new_empty(shape, dtype=torch.float32), hidden.new_empty((16 + 5 * targets.numel(),), dtype=torch.float32)]
    # whole numbers: symbolic sizes are fixed here, as they decide how many tensors there are
    size = unit_elements(int(targets.numel()), int(weight.shape[0]), int(weight.shape[1]), dtype_code(weight), gradients)
    return [*res, hidden.new_empty((size,), dtype=torch.float32)] if size else res


def run_head_logps(hidden, weight, targets, ignore_index, temperature, gradients):
    out = torch.empty(targets.shape, dtype=torch.float32, device=targets.device)
    return _forward("me_head_logps", hidden, weight, targets, ignore_index, gradients, out, (temperature,))


@_custom_op("head_logps")
def head_logps(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, ignore_index: int,
               temperature: float, gradients: int) -> List[torch.Tensor]:
    """[log-probabilities fp32 of targets' shape, saved (what the backward needs)], and where unit_elements says so unit: bf16,
    what the backward of hidden alone only scales; few rows of fp32, their logits."""
    return run_head_logps(hidden, weight, targets, ignore_index, temperature, gradients)[0]


@head_logps.register_fake
def _(hidden, weight, targets, ignore_index, temperature, gradients):
    return _fake_forward(hidden, weight, targets, gradients, targets.shape)


def run_head_ce(hidden, weight, targets, ignore_index, temperature, smoothing, z_loss, scale, reduction, gradients):
    out = torch.empty((), dtype=torch.float32, device=targets.device)
    return _forward("me_head_ce", hidden, weight, targets, ignore_index, gradients, out,
                    (temperature, smoothing, z_loss, scale, reduction))


@_custom_op("head_ce")
def head_ce(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, ignore_index: int, temperature: float,
            smoothing: float, z_loss: float, scale: float, reduction: int, gradients: int) -> List[torch.Tensor]:
    """[loss fp32, saved], and unit as of head_logps."""
    return run_head_ce(hidden, weight, targets, ignore_index, temperature, smoothing, z_loss, scale, reduction, gradients)[0]


@head_ce.register_fake
def _(hidden, weight, targets, ignore_index, temperature, smoothing, z_loss, scale, reduction, gradients):
    return _fake_forward(hidden, weight, targets, gradients, ())


@_custom_op("head_backward")
def head_backward(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, saved: torch.Tensor,
                  unit: Optional[torch.Tensor], upstream: torch.Tensor, ignore_index: int, temperature: float, per_row: bool,
                  smoothing: float, z_loss: float, scale: float, reduction: int, need_hidden: bool,
                  need_weight: bool) -> List[torch.Tensor]:
    """The gradients that are needed, of hidden and of weight. upstream: fp32, one (head_ce) or per row (head_logps)."""
    require_gpu(hidden, weight, targets, saved, unit, upstream)
    _, operands = held = _operands(hidden, weight, targets, ignore_index)
    grads = _backward(hidden.shape, weight.shape, operands, hidden, saved, unit, upstream,
                      (temperature, per_row, smoothing, z_loss, scale, reduction), need_hidden, need_weight)
    del held  # the operands are addresses in these
    return [g for g in grads if g is not None]


@head_backward.register_fake
def _(hidden, weight, targets, saved, unit, upstream, ignore_index, temperature, per_row, smoothing, z_loss, scale,
      reduction, need_hidden, need_weight):
    return [x.new_empty(x.shape) for x, need in ((hidden, need_hidden), (weight, need_weight)) if need]
