"""Operators on a decoder's logits: what it answers with, and what it learns from.

Each case is one call that a user's program makes on logits [rows, vocabulary]:

  sample   ``kvm_amd.sample_tokens``: the next token of every sequence under a
           temperature, top-k, top-p and min-p, from given uniform numbers
  top      ``kvm_amd.top_logits``: a teacher's K largest logits of every
           position with the log-sum-exp of all others, as a distillation keeps them
  distil   ``kvm_amd.distillation_loss`` and its gradient: a student's logits
           against such a teacher, with or without hard labels
  ce       ``kvm_amd.cross_entropy`` and its gradient: a language model's loss

Inputs are synthetic and made from a seed on the GPU: logits of a spread of 2
nats with 40 tokens per row lifted by up to 12, rounded to bfloat16 (what an LM
head writes) and held in the case's type; a teacher whose tokens are among the
lifted ones; labels of which some are ignored (prompt and padding).

Definitions (V logits x of a row, log-sum-exp LSE, all in real arithmetic):

  sample   the tokens in order of falling logit, ties by rising index, have the
           weights w_j = floor(2^42 exp((x_j - x_0) / T) + 1/2); the first top_k
           of them are kept, of these the shortest prefix that holds top_p of
           their weight, of these the tokens with w_j >= min_p 2^42; C_j is the
           running sum of the kept weights and C its end.  The token is the first with
           C_j > floor(u C), its log-probability (x_j - x_0) / T - ln(C 2^-42).
           T = 0 takes the first token, with log-probability 0.
  top      the K largest logits in that same order, their indices, and
           rest = LSE(x_i / T over the other tokens).
  distil   p = softmax over (teacher values / T, rest), q the student's
           probabilities of the same tokens and of all others together at T:
           (1 - a) T^2 sum_k p_k ln(p_k / q_k) + a (LSE(x) - x_label), mean over
           the rows whose label counts.  Without a rest p is the softmax over
           the K values and the sum has their terms alone.
  ce       LSE(x) - x_label, mean over the rows whose label counts.
"""

import functools
import math
import os
import sys
from types import SimpleNamespace

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORE = -100
UNIT = float(1 << 42)  # sampling weights are whole multiples of 2^-42 of the largest


def listed():
    return [
        # One chat sequence: the model's fp32 logits of one token, nucleus sampling.
        dict(name="sample_chat", kind="sample", n=1, V=50304, type="fp32", T=0.8, k=0, p=0.95, m=0.0),
        # A small serving batch: top 50, then a nucleus, as chat servers set by default.
        dict(name="sample_top_k", kind="sample", n=8, V=65536, type="fp32", T=0.7, k=50, p=0.9, m=0.0),
        # A batch of 64 users, each with settings of its own (greedy ones among them), odd vocabulary.
        dict(name="sample_users", kind="sample", n=64, V=50257, type="fp32", T=-1.0, k=0, p=1.0, m=0.0),
        # Rollouts for training: 512 sequences, the model's own distribution with a min-p floor.
        dict(name="sample_rollout", kind="sample", n=512, V=65536, type="bf16", T=1.0, k=0, p=1.0, m=0.02),
        # A teacher that scores one step of 8 sequences.
        dict(name="top_step", kind="top", n=8, V=65536, type="fp32", k=20, T=1.0),
        # A teacher that scores a batch of 8192 positions for a distillation.
        dict(name="top_batch", kind="top", n=8192, V=50304, type="bf16", k=64, T=2.0),
        # The same from fp32 logits of an odd vocabulary, many values kept.
        dict(name="top_odd", kind="top", n=1021, V=50257, type="fp32", k=200, T=1.0),
        # A small student's step on a toy vocabulary: latency counts.
        dict(name="distil_small", kind="distil", n=256, V=1024, type="fp32", k=16, T=1.0, a=0.0, rest=True),
        # A training step of 8192 positions: soft and hard targets.
        dict(name="distil_batch", kind="distil", n=8192, V=50304, type="bf16", k=64, T=2.0, a=0.25, rest=True),
        # fp16 logits of an odd vocabulary, teacher without the mass of the others.
        dict(name="distil_odd", kind="distil", n=2047, V=50257, type="fp16", k=33, T=1.0, a=0.5, rest=False),
        # Pretraining: 2 sequences of 8192 tokens.
        dict(name="ce_batch", kind="ce", n=16384, V=50304, type="bf16"),
        # Fine-tuning on a short sequence with fp32 logits.
        dict(name="ce_short", kind="ce", n=509, V=32000, type="fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = {c["name"]: c for c in listed()}
    while True:
        kind = rng.choice(["sample", "sample", "sample", "top", "top", "distil", "distil", "ce"])
        c = dict(kind=kind, V=rng.choice([32000, 50257, 50304, 65536, _log_int(rng, 600, 131072), _log_int(rng, 600, 131072)]))
        if kind == "sample":
            c.update(n=_log_int(rng, 1, 512), type=rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                     T=rng.choice([-1.0, 0.0, 0.6, 0.8, 1.0, 1.0, 1.3]), k=rng.choice([0, 0, 1, 20, 50, 200, 1000]),
                     p=rng.choice([1.0, 0.95, 0.9, 0.5]), m=rng.choice([0.0, 0.0, 0.05, 0.1]))
            limit = top["sample_rollout"]
        elif kind == "top":
            c.update(n=_log_int(rng, 1, 8192), type=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                     k=min(_log_int(rng, 1, 512), c["V"]), T=rng.choice([1.0, 1.0, 2.0, 4.0]))
            limit = top["top_batch"]
        elif kind == "distil":
            c.update(n=_log_int(rng, 1, 8192), type=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                     k=_log_int(rng, 1, 256), T=rng.choice([1.0, 1.0, 2.0, 4.0]),
                     a=rng.choice([0.0, 0.0, 0.25, 0.5]), rest=rng.choice([True, True, False]))
            limit = top["distil_batch"]
        else:
            c.update(n=_log_int(rng, 1, 16384), type=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
            limit = top["ce_batch"]
        if work(c)["bytes"] <= work(limit)["bytes"]:
            return c


# ---------------------------------------------------------------- inputs

def _logits(g, n, V, kind, lifted):
    """Logits of the given type holding bfloat16 values, tokens ``lifted`` [n, m] raised by up to 12."""
    x = torch.randn(n, V, generator=g, device=DEV).mul_(2.0)
    x.scatter_add_(1, lifted, 12.0 * torch.rand(lifted.shape, generator=g, device=DEV))
    return x.bfloat16().to(TYPES[kind])


def _tokens(g, n, m, V):
    """m different tokens per row, one of each of m equal parts of the vocabulary."""
    at = (torch.arange(m, device=DEV) + torch.rand(n, m, generator=g, device=DEV) * 0.999) * (V / m)
    return at.long().clamp_(max=V - 1)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    n, V = c["n"], c["V"]
    s = SimpleNamespace(case=c)
    if c["kind"] != "distil":
        s.logits = _logits(g, n, V, c["type"], _tokens(g, n, 40, V))
    if c["kind"] == "sample":
        s.u = torch.rand(n, generator=g, device=DEV)
        if c["T"] < 0:  # every row its own settings

            def pick(values, dtype):
                at = torch.randint(0, len(values), (n,), generator=g, device=DEV)
                return torch.tensor(values, device=DEV, dtype=dtype)[at]

            s.T = pick([0.0, 0.5, 0.8, 1.0, 1.0, 1.4], torch.float32)
            s.k = pick([0, 0, 1, 40, 100, 2000], torch.int32)
            s.p = pick([1.0, 0.98, 0.9, 0.7], torch.float32)
            s.m = pick([0.0, 0.0, 0.02, 0.1], torch.float32)
        else:
            s.T, s.k, s.p, s.m = c["T"], c["k"], c["p"], c["m"]
    if c["kind"] == "distil":
        idx = _tokens(g, n, c["k"], V)
        s.logits = _logits(g, n, V, c["type"], idx)
        values = s.logits.gather(1, idx).float() + torch.randn(idx.shape, generator=g, device=DEV)
        s.values = values.bfloat16().to(TYPES[c["type"]])
        s.indices = idx
        s.rest = None
        if c["rest"]:
            s.rest = math.log(V) + 1.0 + torch.randn(n, generator=g, device=DEV)
    if c["kind"] in ("distil", "ce"):
        s.labels = torch.randint(0, V, (n,), generator=g, device=DEV)
        s.labels[torch.rand(n, generator=g, device=DEV) < 0.1] = IGNORE
        if c["kind"] == "distil" and c["a"] == 0:
            s.labels = None
        s.logits.requires_grad_(True)
    return s


# ---------------------------------------------------------------- the plain forms

def _param(v, n, dtype):
    """A setting as a column [n, 1]; plain numbers are held in ``dtype`` first."""
    return (v if isinstance(v, torch.Tensor) else torch.full((n,), v, device=DEV, dtype=dtype)).view(-1, 1)


def _plain_sample(x, u, T, k, p, m):
    n, V = x.shape
    T, p, m = (_param(v, n, torch.float32).double() for v in (T, p, m))
    k = _param(k, n, torch.int64).long()
    values, order = x.float().sort(dim=-1, descending=True, stable=True)
    d = values.double() - values[:, :1].double()
    greedy = T <= 0
    w = torch.floor(torch.exp(d / torch.where(greedy, 1.0, T)) * UNIT + 0.5).long()
    rank = torch.arange(V, device=DEV)
    w = torch.where((rank < torch.where(k <= 0, V, k)) & (~greedy | (rank == 0)), w, 0)
    run_ = w.cumsum(-1)
    keep = ((run_ - w).double() < p * run_[:, -1:].double()) & (w.double() >= m * UNIT)
    run_ = torch.where(keep | (rank == 0), w, 0).cumsum(-1)
    total = run_[:, -1:].double()
    at = torch.floor(u.double().view(-1, 1) * total).long()
    j = (run_ <= at).sum(-1, keepdim=True)
    logprob = d.gather(1, j) / torch.where(greedy, 1.0, T) - torch.log(total / UNIT)
    return order.gather(1, j).squeeze(1), torch.where(greedy, 0.0, logprob).float().squeeze(1)


def _lse(x):
    top = x.max(-1, keepdim=True).values
    return top.squeeze(-1) + torch.log(torch.exp(x - top).sum(-1))


def _plain_top(x, k, T):
    V = x.shape[1]
    xf = x.float()
    bits = xf.view(torch.int32).long()
    key = torch.where(bits < 0, -1 - (bits & 0x7FFFFFFF), bits)  # ordered as the floats are
    key = (key << 20) + (V - 1 - torch.arange(V, device=DEV))      # ties by rising index
    idx = key.topk(k, dim=-1).indices
    rest = _lse(xf.scatter(1, idx, -math.inf) / T) if k < V else torch.full_like(xf[:, 0], -math.inf)
    return x.gather(1, idx), idx, rest


def _plain_targets(xf, labels, n):
    counted = torch.ones(n, device=DEV, dtype=torch.bool) if labels is None else labels != IGNORE
    return counted, counted.sum().clamp(min=1)


def _plain_ce_rows(xf, labels, counted):
    """Row losses LSE(x) - x_label and their gradients."""
    at = torch.where(counted, labels, 0).view(-1, 1)
    lse = _lse(xf)
    grad = torch.exp(xf - lse.view(-1, 1))
    grad.scatter_add_(1, at, torch.full_like(xf[:, :1], -1.0))
    return lse - xf.gather(1, at).squeeze(1), grad


def _plain_distil_rows(xf, values, idx, rest, T):
    """Row losses T^2 KL and their gradients."""
    z = xf / T
    t = values.double() / T
    if rest is not None:
        t = torch.cat([t, rest.double().view(-1, 1)], 1)
    logp = t - _lse(t).view(-1, 1)
    p = torch.exp(logp)
    lse = _lse(z).view(-1, 1)
    logq = z.gather(1, idx).double() - lse.double()
    grad = torch.exp(z - lse)
    if rest is not None:
        zr = z.scatter(1, idx, -math.inf)
        lr = _lse(zr).view(-1, 1)
        logq = torch.cat([logq, (lr - lse).double()], 1)
        grad -= p[:, -1:].float() * torch.exp(zr - lr)
    grad.scatter_add_(1, idx, -p[:, :idx.shape[1]].float())
    return T * T * (p * (logp - logq)).sum(-1).float(), grad.mul_(T)


def _plain_loss(s):
    c, x = s.case, s.logits.detach()
    xf = x.float()
    counted, count = _plain_targets(xf, s.labels, c["n"])
    if c["kind"] == "ce":
        loss, grad = _plain_ce_rows(xf, s.labels, counted)
    else:
        loss, grad = _plain_distil_rows(xf, s.values, s.indices, s.rest, c["T"])
        if c["a"]:
            hard, hard_grad = _plain_ce_rows(xf, s.labels, counted)
            loss = (1 - c["a"]) * loss + c["a"] * hard
            grad = grad.mul_(1 - c["a"]).add_(hard_grad, alpha=c["a"])
    scale = counted.float() / count
    return (loss * scale).sum(), grad.mul_(scale.view(-1, 1)).to(x.dtype)


# ---------------------------------------------------------------- one pass

@functools.lru_cache(None)
def _framework():
    sys.path.insert(0, os.path.join(os.getcwd(), "kvm-paper_amd"))
    import kvm_amd

    return kvm_amd


def run(s):
    c = s.case
    if own:
        fw = _framework()
        if c["kind"] == "sample":
            return fw.sample_tokens(s.logits, s.u, temperature=s.T, top_k=s.k, top_p=s.p, min_p=s.m,
                                    return_logprobs=True)
        if c["kind"] == "top":
            t = fw.top_logits(s.logits, c["k"], temperature=c["T"])
            return t.values, t.indices, t.rest
        if c["kind"] == "distil":
            teacher = fw.TopLogits(s.values, s.indices, s.rest, c["T"])
            loss = fw.distillation_loss(s.logits, teacher, s.labels, label_weight=c["a"])
        else:
            loss = fw.cross_entropy(s.logits, s.labels)
        return loss.detach(), torch.autograd.grad(loss, s.logits)[0]
    if c["kind"] == "sample":
        return _plain_sample(s.logits, s.u, s.T, s.k, s.p, s.m)
    if c["kind"] == "top":
        return _plain_top(s.logits, c["k"], c["T"])
    return _plain_loss(s)


def work(case):
    """Each input read once, each output written once; an exponential and its sum (two for soft targets beside hard ones)
    count four operations, a gradient's value two more."""
    c = case
    size = 4.0 if c["type"] == "fp32" else 2.0
    values = float(c["n"]) * c["V"]
    if c["kind"] == "sample":
        return {"bytes": size * values + c["n"] * (4.0 + 8.0 + 4.0), "flops": 4 * values}
    if c["kind"] == "top":
        return {"bytes": size * values + c["n"] * (c["k"] * (size + 8.0) + 4.0), "flops": 4 * values}
    if c["kind"] == "distil":
        return {"bytes": 2 * size * values + c["n"] * (c["k"] * (size + 8.0) + 4.0 * c["rest"] + 8.0 * (c["a"] > 0)) + 4,
                "flops": (6 + (4 if c["a"] > 0 and c["T"] != 1 else 0)) * values}
    return {"bytes": 2 * size * values + 8.0 * c["n"] + 4, "flops": 6 * values}


# ---------------------------------------------------------------- 64 bits

def _exact_sample(x, u, T, k, p, m):
    """Row by row, on sorted whole-number weights."""
    n, V = x.shape
    get = lambda v, i: float(v[i]) if isinstance(v, torch.Tensor) else float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
    tokens, logprobs = [], []
    for i in range(n):
        row = x[i].double()
        best = row.max()
        t = get(T, i)
        if t <= 0:
            tokens.append((row == best).nonzero()[0, 0])
            logprobs.append(torch.zeros((), device=DEV, dtype=torch.float64))
            continue
        w = (torch.exp((row - best) / t) * UNIT + 0.5).floor().long()
        order = torch.argsort(-row, stable=True)
        kept = order if int(get(k, i)) <= 0 else order[:int(get(k, i))]
        before = w[kept].cumsum(0) - w[kept]
        kept = kept[before.double() < get(p, i) * w[kept].sum().double()]
        strong = kept[w[kept].double() >= get(m, i) * UNIT]
        kept = strong if strong.numel() else kept[:1]
        ends = w[kept].cumsum(0)
        target = (u[i].double() * ends[-1].double()).floor().long()
        token = kept[torch.searchsorted(ends, target, right=True)]
        tokens.append(token)
        logprobs.append((row[token] - best) / t - torch.log(ends[-1].double() / UNIT))
    return torch.stack(tokens), torch.stack(logprobs)


def exact(case, seed):
    c = dict(case)
    s = prepare(case, seed)
    if c["kind"] == "sample":
        return _exact_sample(s.logits, s.u, s.T, s.k, s.p, s.m)
    if c["kind"] == "top":
        x = s.logits.double()
        order = torch.argsort(-x, dim=-1, stable=True)
        top, others = order[:, :c["k"]], order[:, c["k"]:]
        return s.logits.gather(1, top), top, torch.logsumexp(x.gather(1, others) / c["T"], -1)
    x = s.logits.detach().double().requires_grad_(True)
    counted = torch.ones(c["n"], device=DEV, dtype=torch.bool) if s.labels is None else s.labels != IGNORE
    loss = 0.0
    if s.labels is not None:
        a = c.get("a", 1.0)
        loss = a * torch.nn.functional.cross_entropy(x, s.labels, ignore_index=IGNORE, reduction="none")
    if c["kind"] == "distil":
        T = c["T"]
        teacher = s.values.double() / T
        student = torch.log_softmax(x / T, -1)
        logq = student.gather(1, s.indices)
        if s.rest is not None:
            teacher = torch.cat([teacher, s.rest.double().view(-1, 1)], 1)
            others = torch.logsumexp(student.scatter(1, s.indices, -math.inf), -1, keepdim=True)
            logq = torch.cat([logq, others], 1)
        logp = torch.log_softmax(teacher, -1)
        loss = loss + (1 - c["a"]) * T * T * (logp.exp() * (logp - logq)).sum(-1)
    loss = torch.where(counted, loss, 0.0).sum() / counted.sum().clamp(min=1)
    return loss.detach(), torch.autograd.grad(loss, x)[0]
