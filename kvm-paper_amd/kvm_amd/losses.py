"""Losses on a decoder's logits, with their gradients (``kvm_head_loss``).

``cross_entropy`` with hard labels, ``distillation_loss`` from a teacher's top
logits (``logits.top_logits``), alone or beside hard labels.  Logits are
bfloat16, float16 or float32 ROCm device tensors [..., V] in the layouts
``logits.py`` names; statistics and losses are float32, and the gradient has
the logits' type.

The forward computes the gradient for an upstream gradient of one while it
holds a row's logits in registers: a training step moves them once in and
their gradient once out.  The backward hands that gradient out, multiplied in
place where the upstream gradient is not one; in float16, whose small numbers
end at 2^-24, it is computed again with the factor in it, so that a scaled loss
keeps what the scale is for.  Calling backward again on a
retained graph computes it again.  The losses are differentiable once.

A step may be captured into a HIP graph, with its backward or either alone (the
backward then hands out a copy).  As for any backward that torch accumulates
into leaves, no graph of eager steps on the same leaves may be alive while it is
captured: torch would accumulate on that graph's stream, outside the capture.
"""

from __future__ import annotations

import torch

from . import _lib
from .logits import TopLogits

_REDUCTIONS = {"mean": 0, "sum": 1, "none": 2}


def _reduction(name: str) -> int:
    if name not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(_REDUCTIONS)}, got {name!r}")
    return _REDUCTIONS[name]


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
    return _lib.call_op(_lib.ops().head_loss, logits, labels, None, None, None, 1.0, 1.0, ignore_index,
                        _reduction(reduction))


def distillation_loss(logits: torch.Tensor, teacher: TopLogits, labels: torch.Tensor | None = None, *,
                      label_weight: float = 0.0, ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """(1 - label_weight) T^2 KL(teacher || student) + label_weight (cross-entropy
    with ``labels``) of every row of a student's ``logits`` [..., V], float32.

    T is the teacher's temperature.  The divergence is between distributions
    over K + 1 outcomes: the teacher's K tokens (at most 1024), and all other
    tokens together (weight ``teacher.rest``).  Without a rest the K values are
    the teacher's whole distribution.  Teacher entries whose index is outside
    the vocabulary are padding, and entries of the same token add up; a row
    with nothing but padding has no soft term.  No gradient flows to the
    teacher.

    ``labels`` [...]: rows with ``ignore_index`` are left out of both terms (a
    mask even where ``label_weight`` is 0); reduction as in
    :func:`cross_entropy`."""
    if teacher is None:
        raise ValueError("distillation_loss needs a teacher")
    values, indices, rest, temperature = TopLogits(*teacher)
    return _lib.call_op(_lib.ops().head_loss, logits, labels, values, indices, rest, float(temperature),
                        float(label_weight), ignore_index, _reduction(reduction))


__all__ = ["cross_entropy", "distillation_loss"]
