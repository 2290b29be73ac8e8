"""Distillation from a teacher's top logits.

Per row, with ``p`` the teacher's softmax over the ``K`` logits it gives and
``q`` the student's over the whole vocabulary, both at a temperature:
``loss = temperature^2 * sum_k p_k (log p_k - log q_{i_k})``.

On CUDA one sm_100a kernel per row (``csrc/bssm_distill.cu``) reads the logits
and, where the loss is reduced to one number, writes their gradient in the same
launch, so a training step reads the logits once and writes the gradient once;
on CPU the formula runs as PyTorch operations.
"""
from __future__ import annotations

import math
from numbers import Real

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _capi
from .selective import _DTYPES, _carries_tangent, _empty_like, _gradients_wanted, _rows

MAX_TOP = 1024


def distillation_loss_torch(logits: Tensor, teacher_logits: Tensor, teacher_indices: Tensor, *,
                            temperature: float = 1.0, reduction: str = "mean") -> Tensor:
    """:func:`distillation_loss` in PyTorch operations, computed in float32
    (float64 for float64 logits)."""
    wide = torch.promote_types(logits.dtype, torch.float32)
    live = (teacher_indices >= 0) & (teacher_logits != -math.inf)
    counted = live.any(-1)
    t = torch.where(live, teacher_logits.to(wide) / temperature, -math.inf)
    t = torch.where(counted[..., None], t, 0.0)
    log_p = torch.log_softmax(t, -1)
    p = torch.where(live, torch.exp(log_p), 0.0)
    bad = (live & (teacher_indices >= logits.shape[-1])).any(-1)
    index = teacher_indices.long().clamp(0, logits.shape[-1] - 1)
    # NaN by a factor, so that the gradient of a row with an entry past the vocabulary is NaN too
    s = torch.where(counted[..., None], logits.to(wide), 0.0) * torch.where(bad, math.nan, 1.0).to(wide)[..., None]
    log_q = torch.gather(torch.log_softmax(s / temperature, -1), -1, index)
    # an entry of no weight adds nothing, whatever its logarithms
    term = torch.where(p != 0, p * (log_p - torch.where(p != 0, log_q, 0.0)), 0.0)
    rows = torch.where(counted, term.sum(-1) * temperature * temperature, 0.0)
    if reduction == "none":
        return rows
    total = rows.sum()
    return total / counted.sum().clamp(min=1) if reduction == "mean" else total


def _forward(logits, teacher, indices, temperature, reduction, with_grad):
    """Loss (of every row, or reduced), its gradient where it is wanted and
    known up to a factor, and what the backward needs otherwise."""
    dev = logits.device
    vocab, top = logits.shape[-1], teacher.shape[-1]
    rows = teacher.numel() // top
    x, stride = _rows(logits, 1)
    mean, reduced = reduction == "mean", reduction != "none"
    # statistics (2 floats a row), row losses, partial counts
    scratch = torch.empty(3 * rows + _capi.load().bssm_distillation_counters(), device=dev, dtype=torch.float32)
    at = scratch.data_ptr()
    loss = torch.empty(() if reduced else logits.shape[:-1], device=dev, dtype=torch.float32)
    grad = _empty_like(logits) if with_grad and reduced else None
    _capi.launch(dev, "bssm_distillation", x.data_ptr(), _DTYPES[x.dtype], rows, vocab, stride, teacher.data_ptr(),
                 _DTYPES[teacher.dtype], indices.data_ptr(), indices.element_size(), top, temperature, mean,
                 at + 8 * rows if reduced else loss.data_ptr(), at, loss.data_ptr() if reduced else None,
                 at + 12 * rows, _capi.ptr(grad))
    return loss, grad, scratch


class _Distillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher, indices, temperature, reduction):
        # the gradient is saved with the rest, so that recomputation and offloading take it along
        loss, grad, scratch = _forward(logits, teacher, indices, temperature, reduction, True)
        ctx.save_for_backward(logits, teacher, indices, scratch, grad)
        ctx.unused = grad is not None
        ctx.settings = (temperature, reduction)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        logits, teacher, indices, scratch, grad = ctx.saved_tensors
        temperature, reduction = ctx.settings
        dev = logits.device
        upstream = upstream.float().contiguous()
        x, stride = _rows(logits, 1)
        top = teacher.shape[-1]
        rows = teacher.numel() // top
        at = scratch.data_ptr()
        flat = (x.data_ptr(), _DTYPES[x.dtype], rows, logits.shape[-1], stride, teacher.data_ptr(),
                _DTYPES[teacher.dtype], indices.data_ptr(), indices.element_size(), top, temperature,
                reduction == "mean", at, at + 12 * rows, upstream.data_ptr())
        # The gradient written by the forward is handed out once, as it is where the upstream one is 1 and computed
        # again where not (the factor comes before the rounding); a second walk through a retained graph makes its own.
        if ctx.unused:
            ctx.unused = False
            grad = grad.data  # with a version of its own: its owner may change it while the graph is retained
            _capi.launch(dev, "bssm_distillation_rescale", *flat, grad.data_ptr())
        else:
            grad = _empty_like(logits)
            _capi.launch(dev, "bssm_distillation_backward", *flat, reduction == "none", grad.data_ptr())
        return grad, None, None, None, None


def distillation_loss(logits: Tensor, teacher_logits: Tensor, teacher_indices: Tensor, *, temperature: float = 1.0,
                      reduction: str = "mean") -> Tensor:
    """``temperature^2 * KL(teacher || student)`` over a teacher's top logits.

    ``logits`` are the student's ``[..., V]``; ``teacher_logits [..., K]`` the
    teacher's logits at vocabulary entries ``teacher_indices [..., K]`` (int32
    or int64).  An entry with a negative index or a logit of ``-inf`` is empty;
    a row of empty entries (a prompt's, or padding) has loss and gradient zero
    and does not count in a mean.  An index at or past V, or a teacher's logit
    of NaN or ``+inf``, makes the row's loss and gradient NaN.  ``reduction``
    is ``"mean"`` (over the rows that count; zero if none does), ``"sum"`` or
    ``"none"`` (``[...]``).  The loss is float32; gradients flow to ``logits``
    only.  CUDA takes up to 1,024 teacher logits a row.
    """
    if logits.ndim < 1 or teacher_logits.ndim != logits.ndim or teacher_logits.shape[:-1] != logits.shape[:-1]:
        raise ValueError("teacher_logits must be [..., K] with the logits' leading dimensions")
    if teacher_indices.shape != teacher_logits.shape:
        raise ValueError("teacher_indices must have the teacher_logits' shape")
    if logits.shape[-1] < 1 or teacher_logits.shape[-1] < 1:
        raise ValueError("logits and teacher_logits must not be empty")
    if not logits.is_floating_point() or not teacher_logits.is_floating_point():
        raise TypeError("logits and teacher_logits must have floating-point dtype")
    if teacher_indices.dtype not in (torch.int32, torch.int64):
        raise TypeError("teacher_indices must be int32 or int64")
    if teacher_logits.device != logits.device or teacher_indices.device != logits.device:
        raise ValueError("logits, teacher_logits and teacher_indices must be on the same device")
    if isinstance(temperature, bool) or not isinstance(temperature, Real) or not math.isfinite(temperature) \
            or temperature <= 0:
        raise ValueError("temperature must be finite and positive")
    if reduction not in ("mean", "sum", "none"):
        raise ValueError("reduction must be 'mean', 'sum' or 'none'")
    if not logits.is_cuda:
        return distillation_loss_torch(logits, teacher_logits.detach(), teacher_indices, temperature=temperature,
                                       reduction=reduction)
    if logits.dtype not in _DTYPES or teacher_logits.dtype not in _DTYPES:
        raise TypeError("distillation_loss on CUDA takes float32, bfloat16 or float16 logits")
    if teacher_logits.shape[-1] > MAX_TOP:
        raise NotImplementedError(f"distillation_loss on CUDA needs at most {MAX_TOP} teacher logits a row "
                                  f"(got {teacher_logits.shape[-1]}); use distillation_loss_torch")
    teacher, indices = teacher_logits.detach().contiguous(), teacher_indices.contiguous()
    if _gradients_wanted(logits) or _carries_tangent(logits):
        return _Distillation.apply(logits, teacher, indices, float(temperature), reduction)
    return _forward(logits, teacher, indices, float(temperature), reduction, False)[0]


__all__ = ["distillation_loss", "distillation_loss_torch"]
