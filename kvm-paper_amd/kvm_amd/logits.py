"""Operators on a decoder's logits: the next token, and a teacher's top logits.

``sample_tokens`` draws the next token of every row under a temperature,
top-k, top-p and min-p from given uniform numbers (``kvm_sample``);
``top_logits`` keeps the K largest logits of every row with the log-sum-exp
of all others (``kvm_top_logits``), which is what ``losses.distillation_loss``
learns from.  Both run on ROCm device tensors in bfloat16, float16 or float32,
on torch's current stream of the tensor's device (csrc/kvm_logits_ops.cpp);
neither synchronises, and both may be captured into a HIP graph.  Logits are
taken as they lie in memory where the vocabulary is contiguous and the leading
axes collapse to two (any slice of a batch, of positions or of the vocabulary
does); others are copied.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib


class TopLogits(NamedTuple):
    """A teacher's largest logits per position, as ``top_logits`` returns them.

    values [..., K] (logits, any order), indices [..., K] (their tokens; one
    outside the vocabulary is padding), rest [...] float32: the log-sum-exp of
    logit / temperature over all other tokens, or None where it is not known
    (the K values are then taken for the whole distribution)."""

    values: torch.Tensor
    indices: torch.Tensor
    rest: torch.Tensor | None = None
    temperature: float = 1.0


def _setting(v, name: str):
    """(tensor of one value per row, or None; the number of every row) of a setting."""
    if isinstance(v, torch.Tensor):
        if v.dim() or v.is_cuda:
            return v, 0
        v = v.item()
    if not math.isfinite(v):
        raise ValueError(f"{name} must be finite, got {v}")
    return None, v


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                  return_logprobs: bool = False):
    """One token per row of ``logits`` [..., V], from ``uniforms`` [...] in [0, 1).

    The tokens of a row are taken in order of falling logit (equal ones by
    rising index).  ``top_k`` (0: off) keeps the first k of them, ``top_p``
    (1: off) of these the shortest prefix that holds top_p of their
    probability, ``min_p`` (0: off) of these the tokens with at least min_p
    times the largest probability; the first one always stays.  The token is
    the one at which the running probability of those kept passes the row's
    uniform number, so the same numbers give the same tokens.  Probabilities
    are softmax(logits / temperature), counted in units of 2^-42 of the
    largest (a token below half a unit is never drawn).

    ``temperature`` 0 takes the first token.  Each setting is a number or a
    tensor of the rows' shape on the same device (one per request; held in
    float32, top_k in int32), whose values are not checked: a temperature that
    is not positive is 0, a top_k below 1 is off.  A logit of -infinity or NaN
    is never drawn; a row with no other gives token 0 and log-probability NaN.

    Returns int64 tokens [...], with ``return_logprobs`` also the float32
    log-probability of each under the distribution it was drawn from."""
    t, t_all = _setting(temperature, "temperature")
    k, k_all = _setting(top_k, "top_k")
    p, p_all = _setting(top_p, "top_p")
    m, m_all = _setting(min_p, "min_p")
    tokens, logprobs = _lib.call_op(_lib.ops().sample_tokens, logits, uniforms, t, k, p, m, float(t_all),
                                    int(k_all), float(p_all), float(m_all))
    return (tokens, logprobs) if return_logprobs else tokens


def top_logits(logits: torch.Tensor, k: int, *, temperature: float = 1.0) -> TopLogits:
    """The ``k`` largest logits of every row of ``logits`` [..., V], largest
    first, equal ones by rising index, with the log-sum-exp of logit /
    temperature over all other tokens (-infinity where k = V).

    1 <= k <= min(V, 512).  A NaN counts as -infinity.  Returns a
    :class:`TopLogits` of values [..., k] in the logits' type, int64 indices
    [..., k] and rest [...] float32; no gradient flows through it."""
    temperature = float(temperature)
    with torch.no_grad():
        return TopLogits(*_lib.call_op(_lib.ops().top_logits, logits, int(k), temperature), temperature)


__all__ = ["TopLogits", "sample_tokens", "top_logits"]
