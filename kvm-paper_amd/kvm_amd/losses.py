"""Losses on a decoder's logits, with their gradients (``kvm_head_loss``).

``cross_entropy`` with hard labels, ``distillation_loss`` from a teacher's top
logits (``logits.top_logits``), alone or beside hard labels.  Logits are
bfloat16, float16 or float32 ROCm device tensors [..., V] in the layouts
``logits.py`` names; statistics and losses are float32, and the gradient has
the logits' type.

The forward computes the gradient for an upstream gradient of one while it
holds a row's logits in registers: a training step moves them once in and
their gradient once out.  The backward hands that gradient out, multiplied in
place where the upstream gradient is not one (a read of it when it is).
Calling backward again on a retained graph computes it again.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .logits import _DTYPES, TopLogits, logits_rows, on_device

MAX_TEACHER = 1024
_REDUCTIONS = ("mean", "sum", "none")


def _gradient_rows(logits: torch.Tensor, desc: _lib.KvmLogits):
    """A tensor shaped as ``logits`` whose rows start at the same offset modulo
    16 bytes as the logits' rows (the kernel stores it in the chunks it loads),
    with as little padding between them as that takes; and its row strides."""
    V, outer, inner = desc.vocab, desc.outer, desc.inner
    size = logits.element_size()
    n = 16 // size
    gi = V + (desc.s_inner - V) % n if inner > 1 else V
    go = inner * gi + (desc.s_outer - inner * gi) % n if outer > 1 else inner * gi
    offset = desc.data % 16 // size
    buf = torch.empty(offset + outer * go, device=logits.device, dtype=logits.dtype)
    return buf.as_strided((outer, inner, V), (go, gi, 1), offset).view(logits.shape), go, gi


class _Call:
    """One loss: its tensors, checked, and its settings."""

    def __init__(self, logits, labels, teacher, label_weight, ignore_index, reduction):
        if reduction not in _REDUCTIONS:
            raise ValueError(f"reduction must be one of {_REDUCTIONS}, got {reduction!r}")
        logits_rows(logits)  # its checks
        rows = logits.shape[:-1]
        self.reduction, self.ignore_index = reduction, int(ignore_index)
        self.label_weight = float(label_weight)
        self.temperature = 1.0
        if labels is not None:
            if labels.dtype not in (torch.int64, torch.int32):
                raise ValueError(f"labels must be int64 or int32, got {labels.dtype}")
            if labels.shape != rows:
                raise ValueError(f"labels must have the rows' shape {tuple(rows)}, got {tuple(labels.shape)}")
            if labels.device != logits.device:
                raise ValueError("labels must be on the logits' device")
            labels = labels.to(torch.int64).contiguous()
        values = indices = rest = None
        if teacher is not None:
            values, indices, rest, temperature = teacher
            self.temperature = float(temperature)
            if not (self.temperature > 0 and math.isfinite(self.temperature)):
                raise ValueError(f"the teacher's temperature must be positive and finite, got {temperature}")
            if values.dtype not in _DTYPES:
                raise ValueError(f"teacher values must be bfloat16, float16 or float32, got {values.dtype}")
            if indices.dtype not in (torch.int64, torch.int32):
                raise ValueError(f"teacher indices must be int64 or int32, got {indices.dtype}")
            if values.shape[:-1] != rows or indices.shape != values.shape or values.dim() != logits.dim():
                raise ValueError(f"teacher values and indices must have shape {(*rows, 'K')}, got "
                                 f"{tuple(values.shape)} and {tuple(indices.shape)}")
            if not 1 <= values.shape[-1] <= MAX_TEACHER:
                raise ValueError(f"a teacher has 1 to {MAX_TEACHER} values per row, got {values.shape[-1]}")
            if rest is not None and rest.shape != rows:
                raise ValueError(f"the teacher's rest must have the rows' shape {tuple(rows)}, got {tuple(rest.shape)}")
            if any(t is not None and t.device != logits.device for t in (values, indices, rest)):
                raise ValueError("the teacher's tensors must be on the logits' device")
            if not 0.0 <= self.label_weight <= 1.0:
                raise ValueError(f"label_weight must be in [0, 1], got {label_weight}")
            if self.label_weight > 0 and labels is None:
                raise ValueError("label_weight needs labels")
            values, indices = values.detach().contiguous(), indices.to(torch.int64).contiguous()
            if rest is not None:
                rest = rest.detach().to(torch.float32).contiguous()
        self.labels, self.values, self.indices, self.rest = labels, values, indices, rest

    def run(self, logits, want_grad: bool):
        """(loss, gradient or None)."""
        desc, x = logits_rows(logits)
        dev, rows = logits.device, logits.shape[:-1]
        d = _lib.KvmHeadLossDesc()
        d.logits = desc
        if self.labels is not None:
            d.labels, d.ignore_index, d.label_weight = self.labels.data_ptr(), self.ignore_index, self.label_weight
        if self.values is not None:
            d.k, d.t_values, d.t_dtype = self.values.shape[-1], self.values.data_ptr(), _DTYPES[self.values.dtype]
            d.t_indices, d.t_rest = self.indices.data_ptr(), _lib.ptr(self.rest)
        d.temperature = self.temperature
        row_loss = torch.empty(rows, device=dev, dtype=torch.float32)
        d.row_loss = row_loss.data_ptr()
        out = row_loss
        if self.reduction != "none":
            scalars = torch.empty(2, device=dev, dtype=torch.float32)
            out = scalars[0]
            d.loss = scalars.data_ptr()
            if self.reduction == "mean":
                d.inv_count = scalars.data_ptr() + 4
        grad = None
        if want_grad:
            grad, d.g_outer, d.g_inner = _gradient_rows(logits, desc)
            d.grad = grad.data_ptr()
        with on_device(dev):
            _lib.check(_lib.load().kvm_head_loss(ctypes.byref(d), _lib.stream_handle(dev)), "head_loss")
        del x
        return out, grad


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, call):
        loss, ctx.grad = call.run(logits, True)
        ctx.call = call
        ctx.save_for_backward(logits)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, up):
        (logits,) = ctx.saved_tensors
        grad, ctx.grad = ctx.grad, None  # handed out once: what is below may change it
        if grad is None:
            grad = ctx.call.run(logits, True)[1]
        up = up.to(torch.float32).contiguous()
        desc, _ = logits_rows(grad, "gradient")
        with on_device(grad.device):
            _lib.check(_lib.load().kvm_scale_rows(ctypes.byref(desc), up.data_ptr(), 1 if up.dim() else 0,
                                                  _lib.stream_handle(grad.device)), "head_loss backward")
        return grad, None


def _loss(logits, labels, teacher, label_weight, ignore_index, reduction):
    call = _Call(logits, labels, teacher, label_weight, ignore_index, reduction)
    if logits.numel() == 0:  # no rows: an empty loss, or 0, that a graph still reaches
        empty = logits.to(torch.float32).sum(-1)
        return empty if reduction == "none" else empty.sum()
    if torch.is_grad_enabled() and logits.requires_grad:
        return _HeadLoss.apply(logits, call)
    return call.run(logits, False)[0]


def cross_entropy(logits: torch.Tensor, labels: torch.Tensor, *, ignore_index: int = -100,
                  reduction: str = "mean") -> torch.Tensor:
    """logsumexp(x) - x[label] of every row of ``logits`` [..., V], float32.

    ``labels`` [...] (int64 or int32); rows whose label is ``ignore_index``
    have loss 0 and gradient 0, and "mean" divides by the number of the others
    (by 1 where there are none).  Any other label outside the vocabulary makes
    the loss and its row's gradient NaN.  ``reduction``: "mean", "sum" or
    "none" (the row losses [...])."""
    if labels is None:
        raise ValueError("cross_entropy needs labels")
    return _loss(logits, labels, None, 1.0, ignore_index, reduction)


def distillation_loss(logits: torch.Tensor, teacher: TopLogits, labels: torch.Tensor | None = None, *,
                      label_weight: float = 0.0, ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """(1 - label_weight) T^2 KL(teacher || student) + label_weight (cross-entropy
    with ``labels``) of every row of a student's ``logits`` [..., V], float32.

    T is the teacher's temperature.  The divergence is between distributions
    over K + 1 outcomes: the teacher's K tokens, and all other tokens together
    (weight ``teacher.rest``).  Without a rest the K values are the teacher's
    whole distribution.  Teacher entries whose index is outside the vocabulary
    are padding, and entries of the same token add up; a row with nothing but
    padding has no soft term.  No gradient flows to the teacher.

    ``labels`` [...]: rows with ``ignore_index`` are left out of both terms (a
    mask even where ``label_weight`` is 0); reduction as in
    :func:`cross_entropy`."""
    if teacher is None:
        raise ValueError("distillation_loss needs a teacher")
    return _loss(logits, labels, TopLogits(*teacher), label_weight, ignore_index, reduction)


__all__ = ["cross_entropy", "distillation_loss"]
