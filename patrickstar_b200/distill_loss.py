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

from ._lib import (PS_DISTILL_MAX_K, PS_DISTILL_MAX_VOCAB, PS_DTYPE_BF16, PS_DTYPE_F16, PS_DTYPE_F32,
                   PS_REDUCE_MEAN, PS_REDUCE_NONE, PS_REDUCE_SUM, PS_TAIL_BUCKET, PS_TAIL_DROP, DistillProblem,
                   check, lib)

_DTYPES = {torch.float16: PS_DTYPE_F16, torch.bfloat16: PS_DTYPE_BF16, torch.float32: PS_DTYPE_F32}
_TAILS = {"drop": PS_TAIL_DROP, "bucket": PS_TAIL_BUCKET}
_REDUCTIONS = {"none": PS_REDUCE_NONE, "sum": PS_REDUCE_SUM, "mean": PS_REDUCE_MEAN}


def _stream_ptr(device):
    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _like_rows(z):
    """An uninitialised tensor of the shape of ``z`` [rows, vocab] whose rows start at the same offsets from
    16-byte boundaries as those of ``z``, so that a kernel can store what it loaded in whole vectors."""
    rows, vocab = z.shape
    per = 16 // z.element_size()
    ld = vocab + (z.stride(0) - vocab) % per if rows > 1 else vocab
    off = z.data_ptr() % 16 // z.element_size()
    if ld == vocab and off == 0:
        return torch.empty((rows, vocab), dtype=z.dtype, device=z.device)
    return torch.empty(rows * ld + off, dtype=z.dtype, device=z.device).as_strided((rows, vocab), (ld, 1), off)


def _point(problem, z, idx, teacher, mask):
    problem.logits, problem.indices, problem.teacher = z.data_ptr(), idx.data_ptr(), teacher.data_ptr()
    problem.mask = mask.data_ptr() if mask is not None else None
    problem.ld_logits, problem.ld_indices, problem.ld_teacher = z.stride(0), idx.stride(0), teacher.stride(0)
    return problem


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, idx, teacher, mask, problem, scaler):
        dev, rows = z.device, z.shape[0]
        _point(problem, z, idx, teacher, mask)
        f32 = dict(dtype=torch.float32, device=dev)
        row_loss, stats = torch.empty(rows, **f32), torch.empty((rows, 4), **f32)
        reduce = problem.reduction != PS_REDUCE_NONE
        loss = torch.empty((), **f32) if reduce else None
        inv_n = torch.empty(1, **f32) if problem.reduction == PS_REDUCE_MEAN and mask is not None else None
        grad = used = None
        if scaler is not None and rows:
            grad, used = _like_rows(z), torch.empty(1, **f32)
        with torch.cuda.device(dev):
            check(lib.ps_distill_forward(
                C.byref(problem), loss.data_ptr() if reduce else None, row_loss.data_ptr(), stats.data_ptr(),
                inv_n.data_ptr() if inv_n is not None else None, scaler.state_ptr if grad is not None else None,
                grad.data_ptr() if grad is not None else None, grad.stride(0) if grad is not None and rows > 1 else
                z.shape[1], used.data_ptr() if used is not None else None, _stream_ptr(dev)), "ps_distill_forward")
        ctx.save_for_backward(z, idx, teacher, mask, stats, inv_n, used)
        ctx.problem, ctx.grad = problem, grad
        return loss if reduce else row_loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        z, idx, teacher, mask, stats, inv_n, used = ctx.saved_tensors
        rows = z.shape[0]
        _point(ctx.problem, z, idx, teacher, mask)   # saved tensors may come back elsewhere
        # the forward call's gradient is handed out once: what receives it may add to it in place
        grad, ctx.grad = ctx.grad, None
        if grad is None:
            grad, used = _like_rows(z), None
        g = grad_out.to(torch.float32)
        if g.dim() and g.stride(0) not in (0, 1):
            g = g.contiguous()
        with torch.cuda.device(z.device):
            check(lib.ps_distill_backward(
                C.byref(ctx.problem), stats.data_ptr(), inv_n.data_ptr() if inv_n is not None else None, g.data_ptr(),
                g.stride(0) if g.dim() and rows > 1 else 0, used.data_ptr() if used is not None else None,
                grad.data_ptr(), grad.stride(0) if rows > 1 else z.shape[1], _stream_ptr(z.device)),
                "ps_distill_backward")
        return grad, None, None, None, None, None


def _rows(t, width):
    t = t.detach().reshape(math.prod(t.shape[:-1]), width)
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
    of ``logits`` and is rounded once.
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
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError("distillation_loss: temperature must be positive and finite; got %r" % (temperature,))
    if not math.isfinite(weight):
        raise ValueError("distillation_loss: weight must be finite; got %r" % (weight,))
    if logits.dim() < 1 or indices.shape != teacher.shape or indices.shape[:-1] != logits.shape[:-1] \
            or indices.dim() != logits.dim():
        raise ValueError("distillation_loss: logits [..., vocab], indices [..., k] and teacher [..., k] do not fit: "
                         "%s, %s, %s" % (tuple(logits.shape), tuple(indices.shape), tuple(teacher.shape)))
    vocab, k = logits.shape[-1], indices.shape[-1]
    if not 1 <= vocab <= PS_DISTILL_MAX_VOCAB or not 1 <= k <= PS_DISTILL_MAX_K:
        raise ValueError("distillation_loss: 1 to %d vocabulary entries and 1 to %d listed ones; got %d and %d"
                         % (PS_DISTILL_MAX_VOCAB, PS_DISTILL_MAX_K, vocab, k))
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
        if not (torch.is_grad_enabled() and logits.requires_grad):
            scaler = None
    z = logits.reshape(math.prod(logits.shape[:-1]), vocab)
    if z.stride(1) != 1 and vocab > 1:
        z = z.contiguous()
    idx, values = _rows(indices, k), _rows(teacher, k)
    if mask is not None:
        mask = mask.detach().reshape(-1).contiguous()
    problem = DistillProblem(
        rows=z.shape[0], vocab=vocab, k=k, dtype=_DTYPES[z.dtype], index_bytes=idx.element_size(),
        teacher_dtype=_DTYPES[values.dtype], tail=_TAILS[tail], reduction=_REDUCTIONS[reduction],
        temperature=temperature, weight=weight)
    out = _Distill.apply(z, idx, values, mask, problem, scaler)
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
