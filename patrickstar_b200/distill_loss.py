"""Distillation from a teacher's top entries: the loss and its gradient.

A teacher's full distribution over a vocabulary is too much to store; its top
entries, (index, value) pairs for each position, are not.  ``distillation_loss``
takes them and the student's logits, and reads the logits once.  Given the loss
scaler that ``backward`` will go through, it writes the gradient in that same
call, already scaled, so that nothing of it is lost in 16 bits before the
optimizer step divides the scale out again.  No counterpart in the reference.
"""
import ctypes as C
import math

import torch

from ._lib import (PS_DISTILL_MAX_K, PS_DISTILL_MAX_VOCAB, PS_REDUCE_MEAN, PS_REDUCE_NONE, PS_REDUCE_SUM,
                   PS_TAIL_BUCKET, PS_TAIL_DROP, DistillProblem, check, lib)
from .block_fp8 import _DTYPES, _autograd_sees
from .streams import current_device, raw_stream

_TAILS = {"drop": PS_TAIL_DROP, "bucket": PS_TAIL_BUCKET}
_SMALLEST, _LARGEST = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max    # what the C struct holds
_REDUCTIONS = {"none": PS_REDUCE_NONE, "sum": PS_REDUCE_SUM, "mean": PS_REDUCE_MEAN}


def _like_rows(z):
    """An uninitialised tensor of the shape of ``z`` [rows, vocab] whose rows start at the same offsets from
    16-byte boundaries as those of ``z``, so that a kernel can store what it loaded in whole vectors."""
    rows, vocab = z.shape
    per = 16 // z.element_size()
    ld = vocab + (z.stride(0) - vocab) % per if rows > 1 else vocab
    off = z.data_ptr() % 16 // z.element_size()
    if ld == vocab and off == 0:
        return z.new_empty((rows, vocab))
    return z.new_empty(rows * ld + off).as_strided((rows, vocab), (ld, 1), off)


def _point(problem, z, idx, teacher, mask):
    problem.logits, problem.indices, problem.teacher = z.data_ptr(), idx.data_ptr(), teacher.data_ptr()
    problem.mask = mask.data_ptr() if mask is not None else None
    problem.ld_logits, problem.ld_indices, problem.ld_teacher = z.stride(0), idx.stride(0), teacher.stride(0)
    return problem


def _forward(z, idx, teacher, mask, problem, scaler):
    """(loss or row losses, buffer of what backward needs, gradient or None).  The buffer's floats: 1 / rows kept,
    the scale of the gradient, two unused ones, four for each row."""
    dev, rows = z.device, z.shape[0]
    reduce = problem.reduction != PS_REDUCE_NONE
    out = z.new_empty(() if reduce else rows, dtype=torch.float32)
    buf = z.new_empty(4 + (5 if reduce else 4) * rows, dtype=torch.float32)
    grad = _like_rows(z) if scaler is not None and rows else None
    at, o = buf.data_ptr(), out.data_ptr()
    _point(problem, z, idx, teacher, mask)
    with current_device(dev):
        check(lib.ps_distill_forward(
            C.byref(problem), o if reduce else None, at + 16 + 16 * rows if reduce else o, at + 16, at,
            scaler.state_ptr if grad is not None else None, grad.data_ptr() if grad is not None else None,
            grad.stride(0) if grad is not None and rows > 1 else z.shape[1], at + 4, raw_stream(dev)),
            "ps_distill_forward")
    return out, buf, grad


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, idx, teacher, mask, problem, scaler):
        out, buf, ctx.grad = _forward(z, idx, teacher, mask, problem, scaler)
        ctx.save_for_backward(z, idx, teacher, mask, buf)
        ctx.problem = problem
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        z, idx, teacher, mask, buf = ctx.saved_tensors
        rows, at = z.shape[0], buf.data_ptr()
        _point(ctx.problem, z, idx, teacher, mask)   # saved tensors may come back elsewhere
        # the forward call's gradient is handed out once: what receives it may add to it in place
        grad, ctx.grad = ctx.grad, None
        used = at + 4 if grad is not None else None
        if grad is None:
            grad = _like_rows(z)
        g = grad_out if grad_out.dtype == torch.float32 else grad_out.to(torch.float32)
        if g.dim() and g.stride(0) not in (0, 1):
            g = g.contiguous()
        with current_device(z.device):
            check(lib.ps_distill_backward(
                C.byref(ctx.problem), at + 16, at, g.data_ptr(), g.stride(0) if g.dim() and rows > 1 else 0, used,
                grad.data_ptr(), grad.stride(0) if rows > 1 else z.shape[1], raw_stream(z.device)),
                "ps_distill_backward")
        return grad, None, None, None, None, None


def _rows(t, width):
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), width)
    return t if t.stride(1) == 1 or width == 1 else t.contiguous()


def distillation_loss(logits, indices, teacher, *, temperature=1.0, tail="drop", mask=None, reduction="mean",
                      weight=1.0, scaler=None):
    """``weight * temperature**2 * KL(teacher || student)`` over a teacher's listed entries.

    ``logits``   [..., vocab] of the student, float16, bfloat16 or float32 on a CUDA device
    ``indices``  [..., k] int32 or int64: the vocabulary indices of the teacher's entries; -1 lists
                 nothing, an index may be listed twice, any other outside of the vocabulary
                 makes its row's loss and gradient NaN
    ``teacher``  [..., k] the entries' values, float16, bfloat16 or float32; no gradient
    ``tail``     what becomes of the teacher's mass outside of the entries.  "drop": the teacher is
                 ``softmax(teacher / temperature)`` over the entries (``teacher``: logits or
                 log-probabilities).  "bucket": ``teacher`` holds log-probabilities at this
                 temperature, and what they leave of 1 is compared with the student's mass
                 outside of the entries
    ``mask``     [...] bool or uint8: rows that count; the others have loss and gradient 0 and are not read
    ``reduction``  "mean" over the rows that count, "sum", or "none" for [...] losses
    ``scaler``   the ``LossScaler`` or ``DynamicLossScaler`` whose ``backward`` the loss goes through.
                 The gradient is then written in this call, times the current scale; a backward
                 that arrives with another factor computes it anew.  Not with reduction "none"

    The loss is float32, computed from 32-bit exponentials and 64-bit logarithms; the gradient has the type
    of ``logits`` and is rounded once.  A second derivative and forward-mode derivatives are refused.
    """
    for t, name in ((logits, "logits"), (teacher, "teacher")):
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in _DTYPES:
            raise TypeError("distillation_loss: %s must be a CUDA tensor of float16, bfloat16 or float32, got %s" % (
                name, "%s on %s" % (t.dtype, t.device) if isinstance(t, torch.Tensor) else type(t).__name__))
    if not isinstance(indices, torch.Tensor) or indices.dtype not in (torch.int32, torch.int64):
        raise TypeError("distillation_loss: indices must be int32 or int64, got %s"
                        % getattr(indices, "dtype", type(indices).__name__))
    if tail not in _TAILS:
        raise ValueError("distillation_loss: tail must be drop or bucket; got %r" % (tail,))
    if reduction not in _REDUCTIONS:
        raise ValueError("distillation_loss: reduction must be none, sum or mean; got %r" % (reduction,))
    if not _SMALLEST <= temperature <= _LARGEST:
        raise ValueError("distillation_loss: temperature must be positive, finite and normal in 32 bits; got %r"
                         % (temperature,))
    if not abs(weight) <= _LARGEST:
        raise ValueError("distillation_loss: weight must be finite in 32 bits; got %r" % (weight,))
    if logits.dim() < 1 or indices.shape != teacher.shape or indices.shape[:-1] != logits.shape[:-1] \
            or indices.dim() != logits.dim():
        raise ValueError("distillation_loss: logits [..., vocab], indices [..., k] and teacher [..., k] do not fit: "
                         "%s, %s, %s" % (tuple(logits.shape), tuple(indices.shape), tuple(teacher.shape)))
    vocab, k = logits.shape[-1], indices.shape[-1]
    most = PS_DISTILL_MAX_VOCAB // (2 if tail == "bucket" else 1)
    if not 1 <= vocab <= most or not 1 <= k <= PS_DISTILL_MAX_K:
        raise ValueError("distillation_loss: 1 to %d vocabulary entries and 1 to %d listed ones; got %d and %d"
                         % (most, PS_DISTILL_MAX_K, vocab, k))
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8):
            raise TypeError("distillation_loss: mask must be bool or uint8, got %s" % mask.dtype)
        if mask.shape != logits.shape[:-1]:
            raise ValueError("distillation_loss: mask must have shape %s, got %s"
                             % (tuple(logits.shape[:-1]), tuple(mask.shape)))
    for t, name in ((indices, "indices"), (teacher, "teacher"), (mask, "mask")):
        if t is not None and t.device != logits.device:
            raise ValueError("distillation_loss: logits on %s, %s on %s" % (logits.device, name, t.device))
    if teacher.requires_grad and torch.is_grad_enabled():
        raise ValueError("distillation_loss gives no gradient to the teacher: detach it")
    if scaler is not None:
        if reduction == "none":
            raise ValueError("distillation_loss: a scaler goes with one loss, not with reduction none")
        if scaler.device != logits.device:
            raise ValueError("distillation_loss: logits on %s, the scaler on %s" % (logits.device, scaler.device))
    z = _rows(logits, vocab)
    idx, values = _rows(indices, k), _rows(teacher.detach() if teacher.requires_grad else teacher, k)
    if mask is not None:
        mask = mask.reshape(-1).contiguous()
    problem = DistillProblem(None, None, None, None, 0, 0, 0, z.shape[0], vocab, k, _DTYPES[z.dtype], idx.element_size(),
                             _DTYPES[values.dtype], _TAILS[tail], _REDUCTIONS[reduction], temperature, weight)
    if _autograd_sees(z):
        out = _Distill.apply(z, idx, values, mask, problem, scaler)
    else:
        out = _forward(z, idx, values, mask, problem, None)[0]
    return out.view(logits.shape[:-1]) if reduction == "none" else out


class DistillationLoss(torch.nn.Module):
    """``distillation_loss`` with its settings kept; ``forward(logits, indices, teacher, mask=None)``."""

    def __init__(self, temperature=1.0, tail="drop", reduction="mean", weight=1.0, scaler=None):
        super().__init__()
        if tail not in _TAILS:
            raise ValueError("tail must be drop or bucket; got %r" % (tail,))
        if reduction not in _REDUCTIONS:
            raise ValueError("reduction must be none, sum or mean; got %r" % (reduction,))
        self.temperature, self.tail, self.reduction, self.weight = temperature, tail, reduction, weight
        self.scaler = scaler

    def forward(self, logits, indices, teacher, mask=None):
        return distillation_loss(logits, indices, teacher, temperature=self.temperature, tail=self.tail, mask=mask,
                                 reduction=self.reduction, weight=self.weight, scaler=self.scaler)
