"""Operators on a decoder's logits: the next token, and a teacher's top logits.

``sample_tokens`` draws the next token of every row under a temperature,
top-k, top-p and min-p from given uniform numbers (``kvm_sample``);
``top_logits`` keeps the K largest logits of every row with the log-sum-exp
of all others (``kvm_top_logits``), which is what ``losses.distillation_loss``
learns from.  Both run on ROCm device tensors in bfloat16, float16 or float32,
on torch's current stream of the tensor's device; neither synchronises, and
both may be captured into a HIP graph.  Logits are taken as they lie in memory
where the vocabulary is contiguous and the leading axes collapse to two (any
slice of a batch, of positions or of the vocabulary does); others are copied.
"""

from __future__ import annotations

import contextlib
import ctypes
import math
from typing import NamedTuple

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.KVM_BF16, torch.float16: _lib.KVM_F16, torch.float32: _lib.KVM_F32}
MAX_VOCAB = 1 << 20
MAX_TOP_LOGITS = 512


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


def on_device(device: torch.device):
    """A guard that makes ``device`` current for a launch; no work where it is."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def row_layout(shape, strides) -> tuple[int, int, int, int] | None:
    """(outer, inner, outer stride, inner stride) of the rows of a tensor
    [..., V], in the order of its leading axes; None where the vocabulary is
    not contiguous or the leading axes do not collapse to two."""
    if shape[-1] > 1 and strides[-1] != 1:
        return None
    axes: list[tuple[int, int]] = []
    for n, st in zip(shape[:-1], strides[:-1]):
        if n == 1:
            continue
        if axes and axes[-1][1] == n * st:
            axes[-1] = (axes[-1][0] * n, st)
        else:
            axes.append((n, st))
    if len(axes) > 2:
        return None
    (outer, s_outer), (inner, s_inner) = [(1, 0)] * (2 - len(axes)) + axes
    return outer, inner, s_outer, s_inner


def logits_rows(logits: torch.Tensor, name: str = "logits") -> tuple[_lib.KvmLogits, torch.Tensor]:
    """The descriptor of logits [..., V] as rows, and the tensor it points to
    (``logits`` itself unless its layout needs a copy)."""
    code = _DTYPES.get(logits.dtype)
    if code is None:
        raise ValueError(f"{name} must be bfloat16, float16 or float32 (got {logits.dtype})")
    if logits.dim() < 1:
        raise ValueError(f"{name} must have a vocabulary axis")
    if not logits.is_cuda:
        raise RuntimeError(f"{name} must be a ROCm device tensor")
    shape = logits.shape
    V = shape[-1]
    if not 1 <= V <= MAX_VOCAB:
        raise ValueError(f"{name}: the vocabulary must have 1 to {MAX_VOCAB} entries, got {V}")
    layout = row_layout(shape, logits.stride())
    if layout is None:
        logits = logits.contiguous()
        layout = row_layout(shape, logits.stride())
    return _lib.KvmLogits(logits.data_ptr(), code, V, *layout), logits


def _setting(v, name: str, like: torch.Tensor, shape, dtype):
    """(number, None) of a setting for every row, or (0, tensor) of one per row."""
    if isinstance(v, torch.Tensor) and not (v.dim() == 0 and not v.is_cuda):
        if v.dim() and v.shape != shape:
            raise ValueError(f"{name} must be a number or have the rows' shape {tuple(shape)}, got {tuple(v.shape)}")
        if v.device != like.device:
            raise ValueError(f"{name} must be on the logits' device")
        return 0, v.to(dtype).expand(shape).contiguous()
    return (v.item() if isinstance(v, torch.Tensor) else v), None


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
    desc, x = logits_rows(logits)
    shape = logits.shape[:-1]
    if uniforms.shape != shape:
        raise ValueError(f"uniforms must have the rows' shape {tuple(shape)}, got {tuple(uniforms.shape)}")
    if uniforms.device != logits.device:
        raise ValueError("uniforms must be on the logits' device")
    d = _lib.KvmSampleDesc()
    d.logits = desc
    u = uniforms.to(torch.float32).contiguous()
    d.uniforms = u.data_ptr()
    keep = []
    for name, v, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                           ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        number, rows = _setting(v, name, logits, shape, dtype)
        if rows is None:
            if not math.isfinite(number):
                raise ValueError(f"{name} must be finite, got {number}")
            setattr(d, name + "_all", int(number) if name == "top_k" else float(number))
        else:
            keep.append(rows)
            setattr(d, name, rows.data_ptr())
    tokens = torch.empty(shape, device=logits.device, dtype=torch.int64)
    logprobs = torch.empty(shape, device=logits.device, dtype=torch.float32) if return_logprobs else None
    d.tokens = tokens.data_ptr()
    d.logprobs = None if logprobs is None else logprobs.data_ptr()
    if tokens.numel():
        with on_device(logits.device):
            _lib.check(_lib.load().kvm_sample(ctypes.byref(d), _lib.stream_handle(logits.device)), "sample_tokens")
    del keep, x, u
    return (tokens, logprobs) if return_logprobs else tokens


def top_logits(logits: torch.Tensor, k: int, *, temperature: float = 1.0) -> TopLogits:
    """The ``k`` largest logits of every row of ``logits`` [..., V], largest
    first, equal ones by rising index, with the log-sum-exp of logit /
    temperature over all other tokens (-infinity where k = V).

    1 <= k <= min(V, 512).  A NaN counts as -infinity.  Returns a
    :class:`TopLogits` of values [..., k] in the logits' type, int64 indices
    [..., k] and rest [...] float32; no gradient flows through it."""
    desc, x = logits_rows(logits)
    if not 1 <= k <= min(desc.vocab, MAX_TOP_LOGITS):
        raise ValueError(f"k must be in [1, {min(desc.vocab, MAX_TOP_LOGITS)}], got {k}")
    temperature = float(temperature)
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    shape = logits.shape[:-1]
    values = torch.empty(*shape, k, device=logits.device, dtype=logits.dtype)
    indices = torch.empty(*shape, k, device=logits.device, dtype=torch.int64)
    rest = torch.empty(shape, device=logits.device, dtype=torch.float32)
    if rest.numel():
        with on_device(logits.device):
            _lib.check(_lib.load().kvm_top_logits(ctypes.byref(desc), k, temperature, values.data_ptr(),
                                                  indices.data_ptr(), rest.data_ptr(),
                                                  _lib.stream_handle(logits.device)), "top_logits")
    del x
    return TopLogits(values, indices, rest, temperature)


__all__ = ["TopLogits", "sample_tokens", "top_logits"]
