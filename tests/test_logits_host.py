"""CPU tests of the operators on logits: refusals before any GPU work, and the 64-bit oracle itself against torch and finite differences."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import logits_oracle as O


def _lib():
    from kvm_amd import _lib as L

    return L, L.load()


def test_refusals_of_the_c_entry_points():
    L, lib = _lib()
    buf = torch.zeros(64)
    p = buf.data_ptr()
    good = dict(data=p, dtype=L.KVM_F32, vocab=16, outer=1, inner=2, s_outer=0, s_inner=16)

    def refused(rc, text):
        assert rc == L.KVM_EINVAL and text in lib.kvm_last_error().decode(), lib.kvm_last_error()

    def top(k=4, t=1.0, values=p, **kw):
        return lib.kvm_top_logits(ctypes.byref(L.KvmLogits(**{**good, **kw})), k, t, values, p, None, None)

    refused(top(data=None), "must be set")
    refused(top(dtype=3), "type")
    refused(top(vocab=0), "vocab")
    refused(top(vocab=(1 << 20) + 1), "vocab")
    refused(top(outer=0), "rows")
    refused(top(outer=1 << 20, inner=1 << 20), "rows")
    refused(top(data=p + 2), "aligned")
    refused(top(k=0), "k must be")
    refused(top(k=17), "k must be")
    refused(top(k=513, vocab=4096), "k must be")
    refused(top(t=0.0), "temperature")
    refused(top(t=math.inf), "temperature")
    refused(top(values=None), "values")
    refused(lib.kvm_top_logits(None, 1, 1.0, p, p, None, None), "must be set")

    def sample(**kw):
        d = L.KvmSampleDesc(logits=L.KvmLogits(**good), uniforms=p, tokens=p, temperature_all=1.0, top_p_all=1.0)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.kvm_sample(ctypes.byref(d), None)

    refused(sample(uniforms=None), "uniforms")
    refused(sample(tokens=None), "tokens")
    refused(sample(temperature_all=-0.5), "temperature")
    refused(sample(temperature_all=math.nan), "temperature")
    refused(sample(top_k_all=-1), "top_k")
    refused(sample(top_p_all=0.0), "top_p")
    refused(sample(top_p_all=1.5), "top_p")
    refused(sample(min_p_all=-0.1), "min_p")
    refused(sample(min_p_all=1.1), "min_p")
    refused(lib.kvm_sample(None, None), "NULL")

    def loss(**kw):
        d = L.KvmHeadLossDesc(logits=L.KvmLogits(**good), labels=p, row_loss=p, temperature=1.0)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.kvm_head_loss(ctypes.byref(d), None)

    refused(loss(labels=None), "labels, a teacher")
    refused(loss(row_loss=None), "row_loss")
    refused(loss(k=-1), "entries")
    refused(loss(k=1025), "entries")
    refused(loss(k=2), "teacher values")
    teacher = dict(k=2, t_values=p, t_indices=p)
    refused(loss(**teacher, t_dtype=7), "type")
    refused(loss(**teacher, temperature=0.0), "temperature")
    refused(loss(**teacher, label_weight=1.5), "label_weight")
    refused(loss(**teacher, label_weight=0.5, labels=None), "label_weight")
    refused(loss(grad=p), "logits")
    refused(loss(grad=p + 4, g_inner=16), "modulo 16")
    refused(loss(grad=p + 16, g_inner=17), "modulo 16")
    refused(lib.kvm_head_loss(None, None), "NULL")
    refused(lib.kvm_scale_rows(ctypes.byref(L.KvmLogits(**good)), None, 0, None), "factor")


def test_refusals_of_the_python_entry_points():
    import kvm_amd as K

    x, u = torch.zeros(3, 8), torch.zeros(3)
    with pytest.raises(RuntimeError, match="ROCm device"):
        K.sample_tokens(x, u)
    with pytest.raises(RuntimeError, match="ROCm device"):
        K.top_logits(x, 2)
    with pytest.raises(RuntimeError, match="ROCm device"):
        K.cross_entropy(x, torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError, match="bfloat16, float16 or float32"):
        K.sample_tokens(x.double(), u)
    with pytest.raises(ValueError, match="vocabulary axis"):
        K.sample_tokens(torch.zeros(()), u)
    with pytest.raises(ValueError, match="reduction"):
        K.cross_entropy(x, torch.zeros(3, dtype=torch.long), reduction="avg")
    with pytest.raises(ValueError, match="labels"):
        K.cross_entropy(x, None)
    with pytest.raises(ValueError, match="teacher"):
        K.distillation_loss(x, None)


def test_decoder_loss_refusals():
    from kvm_amd import MixerConfig, RWKV7BackboneForCausalLM

    cfg = MixerConfig(vocab_size=32, num_hidden_layers=1, num_attention_heads=1, hidden_size=64, mup_base_dim=64,
                      chunk_len=16, state_min_len=16, rope_partial_dim=32, use_value_residual=0)
    model = RWKV7BackboneForCausalLM(cfg)
    ids = torch.zeros(2, 5, dtype=torch.long)
    with pytest.raises(ValueError, match="labels, a teacher"):
        model.loss(ids)
    with pytest.raises(ValueError, match="shape of input_ids"):
        model.loss(ids, ids[:, :-1])
    with pytest.raises(ValueError, match="uniforms must be"):
        model.generate_sampled(ids, 3, uniforms=torch.zeros(2, 4))


def test_oracle_losses_against_torch_and_differences():
    g = torch.Generator().manual_seed(1)
    n, V, K, T, a = 4, 37, 5, 1.7, 0.3
    x = torch.randn(n, V, generator=g).double()
    idx = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(n)])
    idx[1, 2] = idx[1, 0]  # a token named twice
    idx[2, 3] = -1         # padding
    values, rest = torch.randn(n, K, generator=g), torch.randn(n, generator=g) + 2
    labels = torch.tensor([3, -100, 36, 0])
    for teacher in (None, (values, idx, rest, T), (values, idx, None, T)):
        loss, grad, _, counted = O.loss_rows(x, labels, teacher, a)
        assert counted.tolist() == [True, False, True, True]
        assert loss[1] == 0 and (grad[1] == 0).all()
        if teacher is None:
            want = torch.nn.functional.cross_entropy(x, labels, reduction="none")
            assert torch.allclose(loss, want, rtol=1e-13)
        h = 1e-5
        for j in range(0, V, 4):
            step = torch.zeros(V).double()
            step[j] = h
            up, down = O.loss_rows(x + step, labels, teacher, a)[0], O.loss_rows(x - step, labels, teacher, a)[0]
            # A central difference is off by h^2 / 6 of the third derivative (below 1) and 1e-15 / h of rounding.
            assert ((up - down) / (2 * h) - grad[:, j]).abs().max() < 1e-9


def test_oracle_sampling_frequencies():
    """Over evenly spaced uniforms a token's share is its kept probability
    (settings that float32 holds exactly)."""
    row = torch.tensor([0.3, 2.0, -1.0, 2.0, 0.9, -math.inf])
    us = (torch.arange(2000).double() + 0.5) / 2000
    for kw in ({}, dict(temperature=0.75), dict(top_k=3), dict(top_p=0.75), dict(min_p=0.25),
               dict(top_k=4, top_p=0.625)):
        p = torch.softmax(row.double() / kw.get("temperature", 1.0), 0)
        order = sorted(range(6), key=lambda i: (-float(row[i]), i))
        keep = order[:kw.get("top_k") or 6]
        total, kept, run = sum(float(p[i]) for i in keep), [], 0.0
        for i in keep:
            if run < kw.get("top_p", 1.0) * total - 1e-12 and p[i] >= kw.get("min_p", 0.0) * p.max():
                kept.append(i)
            run += float(p[i])
        share = {i: float(p[i]) / sum(float(p[k]) for k in kept) for i in kept}
        got = [O.sample_row(row, u, **kw) for u in us]
        for i in range(6):
            assert abs(sum(t == i for t, _ in got) / 2000 - share.get(i, 0.0)) <= 1 / 2000
        for t, lp in got[::97]:
            assert abs(lp - math.log(share[t])) < 1e-10
