"""torch custom ops over the head entry points of libmicro_engram_amd.so (csrc/head.hip), in the manner of
loss_ops.py. losses.py is the surface for users.
"""
import ctypes
from typing import List

import torch

from ._lib import call
from .loss_ops import _targets, row_layout
from .ops import _custom_op, call_on, dtype_code, require_gpu


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


def _workspace(hidden, weight, head, n, backward):
    """(buffer, address, size)."""
    size = ctypes.c_size_t(0)
    call("me_head_workspace_size", n, head[1], weight.shape[1], dtype_code(weight), head[0], head[2], backward, ctypes.byref(size))
    ws = torch.empty(size.value, dtype=torch.uint8, device=hidden.device)
    return ws, ws.data_ptr(), ws.numel()


def _forward(name, hidden, weight, targets, ignore_index, out, args):
    dev = require_gpu(hidden, weight, targets)
    held, operands = _operands(hidden, weight, targets, ignore_index)
    n = operands[2]
    saved = torch.empty(16 + 4 * n, dtype=torch.float32, device=dev)
    ws, ptr, size = _workspace(held[0], held[1], operands[7:10], n, 0)
    call_on(dev, name, *operands, *args, out.data_ptr(), saved.data_ptr(), ptr, size)
    return [out, saved]


@_custom_op("head_logps")
def head_logps(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, ignore_index: int,
               temperature: float) -> List[torch.Tensor]:
    """[log-probabilities fp32 of targets' shape, saved (what the backward needs)]."""
    out = torch.empty(targets.shape, dtype=torch.float32, device=targets.device)
    return _forward("me_head_logps", hidden, weight, targets, ignore_index, out, (temperature,))


@head_logps.register_fake
def _(hidden, weight, targets, ignore_index, temperature):
    return [hidden.new_empty(targets.shape, dtype=torch.float32),
            hidden.new_empty((16 + 4 * targets.numel(),), dtype=torch.float32)]


@_custom_op("head_ce")
def head_ce(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, ignore_index: int, temperature: float,
            smoothing: float, z_loss: float, scale: float, reduction: int) -> List[torch.Tensor]:
    """[loss fp32, saved]."""
    out = torch.empty((), dtype=torch.float32, device=targets.device)
    return _forward("me_head_ce", hidden, weight, targets, ignore_index, out,
                    (temperature, smoothing, z_loss, scale, reduction))


@head_ce.register_fake
def _(hidden, weight, targets, ignore_index, temperature, smoothing, z_loss, scale, reduction):
    return [hidden.new_empty((), dtype=torch.float32), hidden.new_empty((16 + 4 * targets.numel(),), dtype=torch.float32)]


@_custom_op("head_backward")
def head_backward(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, saved: torch.Tensor,
                  upstream: torch.Tensor, ignore_index: int, temperature: float, per_row: bool, smoothing: float,
                  z_loss: float, scale: float, reduction: int, need_hidden: bool, need_weight: bool) -> List[torch.Tensor]:
    """The gradients that are needed, of hidden and of weight. upstream: fp32, one (head_ce) or per row (head_logps)."""
    dev = require_gpu(hidden, weight, targets, saved, upstream)
    held, operands = _operands(hidden, weight, targets, ignore_index)
    n = operands[2]
    grad_hidden = torch.empty(hidden.shape, dtype=hidden.dtype, device=dev) if need_hidden else None
    grad_weight = torch.empty(weight.shape, dtype=weight.dtype, device=dev) if need_weight else None
    ws, ptr, size = _workspace(held[0], held[1], operands[7:10], n, 1)
    grads = [g for g in (grad_hidden, grad_weight) if g is not None]
    call_on(dev, "me_head_backward", *operands, temperature, upstream.data_ptr(), int(per_row), smoothing, z_loss, scale,
            reduction, saved.data_ptr(), grad_hidden.data_ptr() if need_hidden else None,
            grad_weight.data_ptr() if need_weight else None, ptr, size)
    return grads


@head_backward.register_fake
def _(hidden, weight, targets, saved, upstream, ignore_index, temperature, per_row, smoothing, z_loss, scale, reduction,
      need_hidden, need_weight):
    return [x.new_empty(x.shape) for x, need in ((hidden, need_hidden), (weight, need_weight)) if need]
