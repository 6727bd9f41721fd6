"""64-bit CPU restatement of the operators on logits: sampling, top logits,
cross-entropy and distillation with their gradients.  Written from the
formulas, row by row."""

from __future__ import annotations

import math

import torch

UNIT = float(1 << 42)


def _clean(row):
    row = row.double()
    return torch.where(row.isnan(), -math.inf, row)


def sample_row(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log-probability) of one row; settings are held in float32."""
    f32 = lambda v: float(torch.tensor(float(v), dtype=torch.float32))  # noqa: E731
    t, p, m = f32(temperature), f32(top_p), f32(min_p)
    row = _clean(row)
    order = torch.sort(-row, stable=True).indices
    best = row[order[0]]
    if best == -math.inf:
        return 0, math.nan
    if not t > 0:
        return int(order[0]), 0.0
    d = torch.where(row[order] == best, 0.0, row[order] - best)  # infinity less itself is no difference
    w = torch.floor(torch.exp(d / t) * UNIT + 0.5).long()
    w[row[order] == -math.inf] = 0
    n = len(row) if top_k <= 0 else min(top_k, len(row))
    w[n:] = 0
    if p < 1:
        before = w.cumsum(0) - w
        w = torch.where(before.double() < p * w.sum().double(), w, 0)
    first = w[0].clone() if w[0] else torch.tensor(int(UNIT))
    if m > 0:
        w = torch.where(w.double() >= m * UNIT, w, 0)
    w[0] = first
    ends = w.cumsum(0)
    target = int(math.floor(min(max(float(u), 0.0), 1.0) * float(ends[-1])))
    j = int(torch.searchsorted(ends, min(target, int(ends[-1]) - 1), right=True))
    return int(order[j]), float(d[j] / t - math.log(float(ends[-1]) / UNIT))


def top_row(row, k, temperature=1.0):
    row = _clean(row)
    order = torch.sort(-row, stable=True).indices
    rest = row[order[k:]] / temperature
    lse = float(torch.logsumexp(rest, 0)) if len(rest) else -math.inf
    return row[order[:k]], order[:k], lse


def _xlogy_terms(p, logp, logq):
    return torch.where(p > 0, p * (logp - logq), torch.zeros_like(p))


def loss_rows(x, labels=None, teacher=None, label_weight=0.0, ignore_index=-100):
    """(row losses [n], row gradients [n, V], size [n, V] of the terms that a
    gradient is the sum of, counted [n]) of logits x [n, V]."""
    x = x.double()
    n, V = x.shape
    a = 1.0 if teacher is None else label_weight
    losses, grads, sizes, counted = [], [], [], []
    for i in range(n):
        row = x[i]
        if row.max().isfinite():
            row = row - row.max()  # nothing below depends on it, and a row of lowest values keeps its digits
        loss, grad, size = torch.zeros((), dtype=torch.float64), torch.zeros(V).double(), torch.zeros(V).double()
        use = labels is None or int(labels[i]) != ignore_index
        counted.append(use)
        if use and teacher is not None and a != 1.0:
            values, idx, rest, T = teacher
            z = row / T
            ok = [k for k in range(idx.shape[1]) if 0 <= int(idx[i, k]) < V]
            t = torch.tensor([float(values[i, k]) / T for k in ok] + ([] if rest is None else [float(rest[i])])).double()
            if rest is not None:
                t[-1] = rest[i].double()
            for q, k in enumerate(ok):
                t[q] = values[i, k].double() / T
            at = torch.tensor([int(idx[i, k]) for k in ok], dtype=torch.long)
            if t.numel() and float(t.max()) > -math.inf:
                t = t - t.max()
                logp = t - torch.logsumexp(t, 0)
                p = logp.exp()
                lse = torch.logsumexp(z, 0)
                named = torch.zeros(V, dtype=torch.bool)
                named[at] = True
                others = torch.where(named, -math.inf, z)
                logq = z[at] - lse
                q = (z - lse).exp()
                g = q.clone()
                s = q.clone()
                if rest is not None:
                    lo = torch.logsumexp(others, 0)
                    logq = torch.cat([logq, (lo - lse).view(1)])
                    if lo > -math.inf:
                        share = p[-1] * (others - lo).exp()
                        g -= share
                        s += share
                P = torch.zeros(V).double().scatter_add(0, at, p[:len(ok)])
                loss = loss + (1 - a) * T * T * _xlogy_terms(p, logp, logq).sum()
                grad = grad + (1 - a) * T * (g - P)
                size = size + (1 - a) * T * (s + P)
        if use and labels is not None and a != 0.0:
            y = int(labels[i])
            if not 0 <= y < V:
                loss, grad = loss * math.nan, grad * math.nan
            else:
                lse = torch.logsumexp(row, 0)
                hot = torch.zeros(V).double()
                hot[y] = 1.0
                loss = loss + a * (lse - row[y])
                grad = grad + a * ((row - lse).exp() - hot)
                size = size + a * ((row - lse).exp() + hot)
        losses.append(loss)
        grads.append(grad)
        sizes.append(size)
    return torch.stack(losses), torch.stack(grads), torch.stack(sizes), torch.tensor(counted)
