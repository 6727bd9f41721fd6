"""Operators on logits (kvm_sample, kvm_top_logits, kvm_head_loss) on the GPU
against the 64-bit oracle of tests/logits_oracle.py.

Bars, from the arithmetic of the kernels:
* tokens, values and indices are equal to the oracle's.  A weight is a whole
  number that two fp64 exponentials round differently only within 2^-50 of a
  half, and a draw could fall on such a unit with a probability below 1e-8.
* a log-probability is an fp64 value rounded to fp32: 2^-24 of it, with the
  absolute 1e-9 that a difference of weights by a unit makes.
* a sum of exponentials in fp32: a thread adds at most 128 terms (2^-24 each,
  7.6e-6 at worst), an exponent of up to 60 log2 units is rounded to 2^-24 of
  itself (60 * 2^-24 * ln 2 = 2.5e-6), the exponential to 1.2e-7, the sums over
  the workgroup add 10 roundings (6e-7): SUM = 1.2e-5 relative, so a logarithm
  of it is off by at most SUM, plus one rounding of the result.
* a gradient is a sum of terms with that relative error, rounded once to its
  type: finfo.eps / 2 of its value, SUM of the size of its terms (each is one
  or two quotients of such sums: 3 SUM), and half the smallest subnormal.
"""

from __future__ import annotations

import math

import pytest
import torch

import kvm_testlib as T
import logits_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
SUM = 1.2e-5
TINY = {torch.bfloat16: 2.0 ** -127, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -127}


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _logits(n, V, dtype, seed, spread=3.0):
    x = torch.randn(n, V, generator=_gen(seed)) * spread
    return x.bfloat16().to(dtype)  # the values an LM head writes, ties among them


# ---------------------------------------------------------------- sampling

def _check_sample(x, u, what, **settings):
    """x [n, V] on the CPU; settings numbers or lists of n."""
    import kvm_amd as K

    T.log(f"[sample] {what} {tuple(x.shape)} {x.dtype} {({k: v for k, v in settings.items() if not isinstance(v, list)})}")
    kinds = dict(temperature=torch.float32, top_k=torch.int32, top_p=torch.float32, min_p=torch.float32)
    dev = {k: torch.tensor(v, dtype=kinds[k], device=DEV) if isinstance(v, list) else v for k, v in settings.items()}
    tok, lp = K.sample_tokens(x.to(DEV), u.to(DEV), **dev, return_logprobs=True)
    tok2 = K.sample_tokens(x.to(DEV), u.to(DEV), **dev)
    assert tok.dtype == torch.int64 and lp.dtype == torch.float32
    tok, lp = tok.cpu(), lp.cpu()
    assert torch.equal(tok, tok2.cpu())
    for i in range(len(x)):
        one = {k: v[i] if isinstance(v, list) else v for k, v in settings.items()}
        wt, wl = O.sample_row(x[i], float(u[i]), **one)
        assert int(tok[i]) == wt, f"row {i}: token {int(tok[i])}, oracle {wt} ({one})"
        if math.isnan(wl):
            assert math.isnan(float(lp[i]))
        else:
            assert abs(float(lp[i]) - wl) <= abs(wl) * 2.0 ** -24 + 1e-9, f"row {i}: {float(lp[i])} {wl}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1, 2, 7, 64, 1000, 4099, 50257])
def test_sample_vocabularies(dtype, V):
    n = 6
    _check_sample(_logits(n, V, dtype, V), torch.rand(n, generator=_gen(V + 1)), "vocabulary")
    _check_sample(_logits(n, V, dtype, V), torch.rand(n, generator=_gen(V + 2)), "nucleus", temperature=0.8, top_p=0.9)
    _check_sample(_logits(n, V, dtype, V), torch.rand(n, generator=_gen(V + 3)), "top-k", top_k=5, top_p=0.7)


@pytest.mark.parametrize("kw", [
    dict(temperature=0.0), dict(top_k=1), dict(temperature=1e-3), dict(temperature=100.0), dict(temperature=1e4),
    dict(top_k=2), dict(top_k=511), dict(top_k=512, min_p=0.01), dict(top_k=513), dict(top_k=2000, top_p=0.5),
    dict(top_k=10 ** 9), dict(top_p=1e-6), dict(top_p=0.999), dict(min_p=1.0), dict(min_p=0.2, temperature=2.0),
    dict(top_k=700, top_p=0.9, min_p=0.05, temperature=1.3), dict(top_k=40, top_p=0.95, min_p=0.05),
    dict(top_p=0.5, min_p=1e-4, temperature=5.0),
])
def test_sample_settings(kw):
    _check_sample(_logits(8, 9001, torch.float32, 5), torch.rand(8, generator=_gen(6)), "settings", **kw)


@pytest.mark.parametrize("kw", [dict(top_k=550), dict(top_k=400, top_p=0.8), dict(top_p=0.97), dict(min_p=0.01),
                                dict(top_p=0.9, min_p=0.02, temperature=3.0), dict(temperature=50.0)])
@pytest.mark.parametrize("V,n", [(600, 4), (700, 300), (2500, 300)])
def test_sample_short_rows_and_many_rows(V, n, kw):
    """Rows that one list of tokens covers, and more rows than compute units."""
    _check_sample(_logits(n, V, torch.bfloat16, V, 1.0), torch.rand(n, generator=_gen(V + n)), "short", **kw)


@pytest.mark.parametrize("kw", [dict(top_p=0.9), dict(top_p=0.6, min_p=0.001), dict(top_k=1500, top_p=0.97),
                                dict(top_k=2000, min_p=0.005), dict(), dict(top_k=2040)])
@pytest.mark.parametrize("spread", [0.02, 0.5, 1.0])
def test_sample_flat_rows(spread, kw):
    """Distributions whose nucleus is hundreds or thousands of tokens."""
    _check_sample(_logits(6, 20011, torch.float32, 77, spread), torch.rand(6, generator=_gen(78)), "flat", **kw)


@pytest.mark.parametrize("n", [9, 270])
@pytest.mark.parametrize("min_p", [0.0, 1e-3])
def test_nucleus_that_ends_on_the_edge_of_a_token(n, min_p):
    """top_p at the running sum of some tokens over the weight of the row, and
    the fp32 numbers beside it: a sum in fp32 does not tell them apart."""
    x = _logits(n, 6007, torch.float32, 79, 3.0)
    w = torch.exp((x.double() - x.max(1, keepdim=True).values.double())).sort(dim=1, descending=True).values
    share = w.cumsum(1) / w.sum(1, keepdim=True)
    p = torch.stack([share[i, (3 * i) % 40] for i in range(n)]).float()
    for step in range(-1, 2):
        at = p if step == 0 else torch.nextafter(p, torch.full_like(p, float(step)))
        _check_sample(x, torch.full((n,), 1.0 - 2.0 ** -24), f"edge {step}", top_p=at.tolist(), min_p=min_p)


@pytest.mark.parametrize("temperature", [1e-39, 1e-30, 1e30, 3e38])
@pytest.mark.parametrize("top_p", [0.7, 1.0])
def test_sample_extreme_temperatures(temperature, top_p):
    x = _logits(5, 5003, torch.float32, 81)
    x[1, :700] = x[1].max() + 1  # ties at the largest value
    x[2, 40] = math.inf
    x[3] = torch.finfo(torch.float32).min
    x[4, ::2] = -math.inf
    _check_sample(x, torch.rand(5, generator=_gen(82)), "extreme", temperature=temperature, top_p=top_p)


def test_sample_settings_per_row():
    n = 24
    g = _gen(9)
    pick = lambda vals: [vals[i] for i in torch.randint(0, len(vals), (n,), generator=g)]  # noqa: E731
    _check_sample(_logits(n, 5003, torch.float32, 8), torch.rand(n, generator=g), "per row",
                  temperature=pick([0.0, 0.5, 1.0, 1.5, -1.0, math.nan]), top_k=pick([0, 1, 30, 900, -5, 10 ** 6]),
                  top_p=pick([1.0, 0.9, 0.3, 0.01]), min_p=pick([0.0, 0.1, 0.9]))


@pytest.mark.parametrize("u", [0.0, 2.0 ** -30, 0.5, 1.0 - 2.0 ** -24, 1.0])
@pytest.mark.parametrize("kw", [dict(), dict(top_p=0.9), dict(top_k=20), dict(min_p=0.1)])
def test_sample_border_uniforms(u, kw):
    _check_sample(_logits(3, 3001, torch.bfloat16, 12), torch.full((3,), u), "border", **kw)


def test_sample_masked_and_degenerate_rows():
    V = 4500
    x = _logits(12, V, torch.float32, 3)
    x[0] = -math.inf                               # nothing left
    x[1] = math.nan                                # nothing but NaN
    x[2, 1:] = -math.inf                           # the first token alone
    x[3, :-1] = -math.inf                          # the last token alone
    x[4] = 0.0                                     # all equal: ties rank by index
    x[5] = -0.0
    x[5, ::2] = 0.0                                # both zeros are equal
    x[6, ::3] = math.nan                           # NaN among numbers
    x[7] = torch.where(torch.rand(V, generator=_gen(4)) < 0.9, torch.finfo(torch.float32).min, x[7])
    x[8, [5, 99, 4000]] = math.inf                 # several infinities share
    x[9] = torch.linspace(0, 1e-4, V)              # clustered: one bin, all different
    x[10] = torch.randn(V, generator=_gen(5)) * 1e30
    x[11] = torch.where(torch.arange(V) % 2 == 0, 1.0, 1.0 + 2.0 ** -20)  # two values, many ties
    for seed, kw in enumerate((dict(), dict(top_p=0.9), dict(top_k=100), dict(top_k=3000, top_p=0.6),
                               dict(min_p=0.5), dict(temperature=0.0))):
        _check_sample(x, torch.rand(12, generator=_gen(20 + seed)), "degenerate", **kw)


def test_sample_large_vocabulary_and_ties():
    V = 150001
    x = _logits(3, V, torch.bfloat16, 31)
    x[1] = 1.0
    x[2] = (torch.randint(0, 3, (V,), generator=_gen(1)).float() * 0.5).bfloat16()
    for kw in (dict(), dict(top_p=0.37), dict(top_k=70000, top_p=0.9), dict(top_k=60)):
        _check_sample(x, torch.rand(3, generator=_gen(2)), "large", **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_largest_vocabulary(dtype):
    V = 1 << 20
    x = _logits(2, V, dtype, 35, 1.5)
    x[1] = x[1].clamp(max=1.0)                     # a tenth of the tokens equal the largest
    for kw in (dict(top_p=0.9), dict(top_k=100), dict()):
        _check_sample(x, torch.tensor([0.3, 0.999]), "largest", **kw)
    _check_top(x, 512, 1.0, "largest")
    _check_loss(x, torch.tensor([V - 1, 5]), _teacher(2, V, 1024, 36, dtype), 0.5, "largest")


def test_sample_views_and_shapes():
    import kvm_amd as K

    base = _logits(6 * 5, 1031, torch.bfloat16, 40).view(6, 5, 1031).to(DEV)
    u = torch.rand(6, 5, generator=_gen(41)).to(DEV)
    for view, uu in ((base[:, :-1], u[:, :-1]), (base[:, -1], u[:, -1]), (base[..., 3:1000], u),
                     (base[1:, 1:, 1:], u[1:, 1:]), (base.transpose(0, 1), u.t()), (base[0, 0], u[0, 0])):
        got = K.sample_tokens(view, uu, top_p=0.9)
        assert got.shape == view.shape[:-1]
        assert torch.equal(got, K.sample_tokens(view.contiguous().clone(), uu.contiguous(), top_p=0.9))
    assert K.sample_tokens(base[:0], u[:0]).shape == (0, 5)


def test_sample_refusals_on_the_gpu():
    import kvm_amd as K

    x, u = torch.zeros(3, 8, device=DEV), torch.zeros(3, device=DEV)
    for kw, text in ((dict(temperature=-1.0), "temperature"), (dict(temperature=math.inf), "finite"),
                     (dict(top_k=-1), "top_k"), (dict(top_p=0.0), "top_p"), (dict(top_p=1.1), "top_p"),
                     (dict(min_p=-0.1), "min_p"), (dict(min_p=2.0), "min_p"),
                     (dict(top_p=torch.ones(2, device=DEV)), "rows' shape"), (dict(top_p=torch.ones(3)), "device")):
        with pytest.raises(ValueError, match=text):
            K.sample_tokens(x, u, **kw)
    with pytest.raises(ValueError, match="uniforms"):
        K.sample_tokens(x, u[:2])
    with pytest.raises(ValueError, match="uniforms"):
        K.sample_tokens(x, u.cpu())
    with pytest.raises(ValueError, match="vocabulary"):
        K.sample_tokens(torch.zeros(3, 0, device=DEV), u)


# ---------------------------------------------------------------- top logits

def _check_top(x, k, temperature, what):
    import kvm_amd as K

    T.log(f"[top] {what} {tuple(x.shape)} {x.dtype} k {k} T {temperature}")
    got = K.top_logits(x.to(DEV), k, temperature=temperature)
    assert got.values.dtype == x.dtype and got.indices.dtype == torch.int64 and got.temperature == temperature
    for i in range(len(x)):
        v, idx, rest = O.top_row(x[i], k, temperature)
        assert torch.equal(got.indices[i].cpu(), idx), f"row {i}"
        assert torch.equal(got.values[i].cpu().double(), v), f"row {i}"
        r = float(got.rest[i])
        if math.isinf(rest):
            assert r == rest, f"row {i}: rest {r}, oracle {rest}"
        else:
            assert abs(r - rest) <= SUM + abs(rest) * 2.0 ** -23, f"row {i}: rest {r}, oracle {rest}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,k", [(1, 1), (5, 5), (5, 2), (300, 299), (1000, 1), (1021, 64), (4100, 512), (40000, 200),
                                 (50257, 20), (140001, 100)])
def test_top_logits_sizes(dtype, V, k):
    _check_top(_logits(4, V, dtype, V + k), k, 1.0 if k % 2 else 2.5, "sizes")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [1, 33, 500])
def test_top_logits_degenerate_rows(dtype, k):
    V = 6007
    x = _logits(11, V, dtype, 50)
    x[0] = -math.inf
    x[1] = math.nan
    x[2] = 0.0                                     # all equal
    x[3] = torch.arange(V)                         # rising: the largest lie side by side
    x[4] = -torch.arange(V).float()
    x[5, 10:] = -math.inf                          # fewer numbers than k
    x[6, ::5] = math.nan
    x[7, [3, 77]] = math.inf
    x[8] = 5.0
    x[8, 1000:1010] = 300.0                        # the others far below
    x[9] = torch.randint(0, 2, (V,), generator=_gen(1)).float()
    x[10] = -0.0
    x[10, ::7] = 0.0
    x[6, 0::9] = torch.finfo(dtype).min
    x[0, :3000] = torch.finfo(dtype).min           # with k = 500: equal lowest values, the others nothing
    x[4, ::2] = torch.arange(V)[::2].remainder(100) * 2.0 ** -133  # subnormal, in order all the same
    _check_top(x, k, 1.0, "degenerate")


def test_top_logits_views_streams_and_refusals():
    import kvm_amd as K

    base = _logits(20, 2003, torch.bfloat16, 60).view(4, 5, 2003).to(DEV)
    for view in (base[:, 1:], base[..., 1:], base[..., 5:1800], base.transpose(0, 1)):
        a, b = K.top_logits(view, 17), K.top_logits(view.contiguous().clone(), 17)
        assert a.values.shape == (*view.shape[:-1], 17)
        assert torch.equal(a.values, b.values) and torch.equal(a.indices, b.indices)
        # Another alignment puts the same terms into other threads' sums: each is within SUM of the true one.
        assert ((a.rest - b.rest).abs() <= 2 * SUM + b.rest.abs() * 2.0 ** -22).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = K.top_logits(base, 9)
    side.synchronize()
    assert torch.equal(c.indices, K.top_logits(base, 9).indices)
    assert K.top_logits(base[:0], 3).indices.shape == (0, 5, 3)
    for k in (0, 513, 2004):
        with pytest.raises(ValueError, match="k must be"):
            K.top_logits(base, k)
    for bad in (0.0, -1.0, math.inf, math.nan, 1e-50, 1e-39):
        with pytest.raises(ValueError, match="temperature"):
            K.top_logits(base, 3, temperature=bad)


# ---------------------------------------------------------------- losses

def _teacher(n, V, k, seed, dtype=torch.float32, temperature=1.0, rest=True):
    g = _gen(seed)
    idx = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(n)])
    values = (torch.randn(n, k, generator=g) * 2).bfloat16().to(dtype)
    return values, idx, torch.randn(n, generator=g) + 1 if rest else None, temperature


def _check_loss(x, labels, teacher, a, what):
    """Row losses, the mean, and the gradients of both against the oracle."""
    import kvm_amd as K

    T.log(f"[loss] {what} {tuple(x.shape)} {x.dtype} K {0 if teacher is None else teacher[1].shape[1]} a {a}")
    want, wgrad, wsize, counted = O.loss_rows(x, labels, teacher, a)
    lab = None if labels is None else labels.to(DEV)
    tch = None if teacher is None else K.TopLogits(*(t.to(DEV) if isinstance(t, torch.Tensor) else t for t in teacher))

    def call(xx, reduction):
        if tch is None:
            return K.cross_entropy(xx, lab, reduction=reduction)
        return K.distillation_loss(xx, tch, lab, label_weight=a, reduction=reduction)

    dev = x.to(DEV)
    kept = dev.clone()
    with torch.no_grad():
        rows = call(dev, "none").cpu().double()
    # The terms of a loss: logarithms of sums (SUM each), in total at most as
    # large as |loss| plus the few nats of the row's own entropies.
    scale = 1.0 if teacher is None else max(1.0, teacher[3] ** 2)
    finite = want.isfinite()
    assert torch.equal(rows.isnan(), want.isnan()) and torch.equal(rows[want.isinf()], want[want.isinf()])
    err = (rows - want).abs()[finite]
    bar = (3 * SUM * scale + want.abs() * 2.0 ** -22)[finite]
    assert (err <= bar).all(), f"row loss off by {err.max():.3g}"
    leaf = dev.clone().requires_grad_(True)
    mean = call(leaf, "mean")
    mean.backward()
    count = max(1, int(counted.sum()))
    if finite.all():
        assert abs(float(mean.detach()) - float(want.sum()) / count) <= 3 * SUM * scale + abs(float(want.sum())) / count * 2.0 ** -22
    g = leaf.grad.cpu().double()
    assert torch.equal(g.isnan(), (wgrad / count).isnan())
    ok = ~wgrad.isnan()
    bar = torch.finfo(x.dtype).eps / 2 * wgrad.abs() / count + 3 * SUM * wsize / count + TINY[x.dtype]
    off = ((g - wgrad / count).abs() - bar)[ok]
    assert (off <= 0).all(), f"gradient over its bar by {off.max():.3g}"
    assert torch.equal(dev, kept) or bool(kept.isnan().any())
    return g


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1, 3, 100, 1000, 4097, 33001])
def test_cross_entropy(dtype, V):
    n = 5
    labels = torch.randint(0, V, (n,), generator=_gen(V))
    labels[1] = -100
    _check_loss(_logits(n, V, dtype, V), labels, None, 1.0, "cross-entropy")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,k,tau,a,rest", [
    (40, 40, 1.0, 0.0, False), (40, 39, 2.0, 0.5, True), (1000, 1, 1.0, 0.0, True), (1003, 16, 2.0, 0.25, True),
    (1003, 16, 2.0, 1.0, True), (5000, 64, 1.0, 0.5, False), (5001, 300, 4.0, 0.0, True), (33001, 1024, 1.5, 0.3, True),
    (150001, 20, 1.0, 0.5, True),
])
def test_distillation(dtype, V, k, tau, a, rest):
    n = 3 if V > 10000 else 5
    labels = torch.randint(0, V, (n,), generator=_gen(V + k)) if a else None
    teacher = _teacher(n, V, k, V, torch.bfloat16 if dtype == torch.float16 else dtype, tau, rest)
    if labels is not None:
        labels[0] = -100
        labels[1] = int(teacher[1][1, 0])  # a label that the teacher names
    _check_loss(_logits(n, V, dtype, V + 7), labels, teacher, a, "distillation")


@pytest.mark.parametrize("tau", [1.0, 2.0])
@pytest.mark.parametrize("rest", [True, False])
def test_distillation_edges(tau, rest):
    n, V, k = 9, 700, 12
    x = _logits(n, V, torch.float32, 70)
    values, idx, r, _ = _teacher(n, V, k, 71, temperature=tau, rest=rest)
    idx[0, 5] = idx[0, 2]
    idx[0, 9] = idx[0, 2]                          # a token three times
    idx[1, 3:] = -1                                # padding
    idx[2] = V                                     # padding only: past the end
    values[3, 2] = -math.inf                       # a token with no probability
    x[4, int(idx[4, 0])] = -math.inf               # the student excludes a likely token: infinite loss
    x[5, 600:] = -math.inf                         # masked vocabulary (the teacher stays below it)
    idx[5] = torch.arange(k)
    x[6] = -200.0
    x[6, idx[6]] = 50.0                            # all other tokens far below
    idx[7] = int(idx[7, 0])                        # one token k times
    x[8, idx[8]] += 100.0 if rest else 30.0
    if rest:
        r[1] = -math.inf                           # the K values are everything
        r[2] = -math.inf                           # an empty teacher
    labels = torch.randint(0, V, (n,), generator=_gen(3))
    labels[0] = int(idx[0, 2])
    labels[5] = 3
    for a in (0.0, 0.4):
        _check_loss(x, labels, (values, idx, r, tau), a, "edges")


def test_label_edges():
    V = 300
    x = _logits(6, V, torch.float32, 80)
    labels = torch.tensor([0, V - 1, V, -1, -100, 7])
    x[5] = torch.finfo(torch.float32).min          # a row of the type's lowest value is flat
    _check_loss(x, labels, None, 1.0, "labels")
    _check_loss(x, labels, _teacher(6, V, 5, 81, temperature=2.0), 0.5, "labels")
    # nothing counts: zero, not a quotient by zero
    g = _check_loss(x, torch.full((6,), -100), None, 1.0, "all ignored")
    assert (g == 0).all()


def test_loss_against_differences():
    """The gradient against central differences of the kernel's own losses:
    h = 0.02 leaves h^2 / 6 of a third derivative below 0.2 T^-1 (1.4e-5), and
    two losses of up to 8, each off by SUM, over 2 h: 6e-4."""
    import kvm_amd as K

    V, h = 29, 0.02
    x = _logits(1, V, torch.float32, 90, 1.0).to(DEV).expand(2 * V, V).clone()
    teacher = K.TopLogits(*(t.to(DEV).expand(2 * V, *t.shape[1:]).contiguous() if isinstance(t, torch.Tensor) else t
                            for t in _teacher(1, V, 6, 91, temperature=1.5)))
    labels = torch.full((2 * V,), 11, device=DEV)
    leaf = x[:1].clone().requires_grad_(True)
    one = K.TopLogits(teacher.values[:1], teacher.indices[:1], teacher.rest[:1], 1.5)
    K.distillation_loss(leaf, one, labels[:1], label_weight=0.4).backward()
    at = torch.arange(V, device=DEV)
    x[at, at] += h
    x[V + at, at] -= h
    rows = K.distillation_loss(x, teacher, labels, label_weight=0.4, reduction="none").double()
    assert ((rows[:V] - rows[V:]) / (2 * h) - leaf.grad[0].double()).abs().max() < 1e-3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_loss_views(dtype):
    """Views of logits give the losses and gradients of their copies, and the
    gradient has the shape of the view."""
    import kvm_amd as K

    base = _logits(4 * 6, 517, dtype, 100).view(4, 6, 517).to(DEV)
    labels = torch.randint(0, 400, (4, 6), generator=_gen(101)).to(DEV)
    for cut in (lambda t: t[:, :-1], lambda t: t[..., 1:], lambda t: t[:, 1:, 2:500], lambda t: t[::2, 3],
                lambda t: t.transpose(0, 1), lambda t: t[1, 2], lambda t: t[:, ::2],
                lambda t: t.transpose(0, 2).contiguous().transpose(0, 2)):  # the vocabulary not contiguous: a copy
        view = cut(base)
        lab = cut(labels.unsqueeze(-1).expand(4, 6, 517))[..., 0].contiguous()
        a = view.detach().requires_grad_(True)
        b = view.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True)
        la, lb = K.cross_entropy(a, lab), K.cross_entropy(b, lab)
        ga, gb = torch.autograd.grad(la, a)[0], torch.autograd.grad(lb, b)[0]
        assert ga.shape == view.shape and torch.equal(la, lb)
        # The same values in other threads: sums differ by their order alone.
        assert ((ga.double() - gb.double()).abs() <= torch.finfo(dtype).eps * gb.double().abs() + 2 * SUM * 0.1).all()


def test_loss_upstream_gradients_and_retained_graphs():
    import kvm_amd as K

    x = _logits(7, 1001, torch.float32, 110).to(DEV).requires_grad_(True)
    labels = torch.randint(0, 1001, (7,), generator=_gen(111)).to(DEV)
    unit = torch.autograd.grad(K.cross_entropy(x, labels, reduction="sum"), x)[0]
    loss = K.cross_entropy(x, labels, reduction="sum")
    first = torch.autograd.grad(2.5 * loss, x, retain_graph=True)[0]
    again = torch.autograd.grad(loss, x, retain_graph=True)[0]
    half = torch.autograd.grad(0.5 * loss, x)[0]
    assert torch.equal(again, unit) and torch.equal(half, 0.5 * unit) and torch.equal(first, 2.5 * unit)
    up = torch.tensor([1.0, 0.0, -2.0, 1.0, 0.25, 3.0, 1.0], device=DEV)
    rows = K.cross_entropy(x, labels, reduction="none")
    got = torch.autograd.grad(rows, x, up)[0]
    assert torch.equal(got, unit * up.view(-1, 1))
    # two losses of one tensor add up in its gradient
    x.grad = None
    (K.cross_entropy(x, labels, reduction="sum") + K.cross_entropy(x, labels, reduction="sum")).backward()
    assert torch.equal(x.grad, 2 * unit)
    with torch.no_grad():
        assert not K.cross_entropy(x, labels).requires_grad
    empty = K.cross_entropy(x[:0], labels[:0])
    assert float(empty.detach()) == 0.0 and K.cross_entropy(x[:0], labels[:0], reduction="none").shape == (0,)
    empty.backward()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("rows,V", [((2, 300), 5003), ((3, 7), 999)])
def test_scaled_losses_keep_small_gradients(dtype, reduction, rows, V):
    """A loss times 2^14 whose unscaled gradient is below fp16's smallest number."""
    import kvm_amd as K

    n = rows[0] * rows[1]
    wide = _logits(n, V + 5, dtype, 115, 1.0).view(*rows, V + 5)
    labels = torch.randint(0, V, rows, generator=_gen(116))
    labels[0, 3] = -100
    x = wide.to(DEV).requires_grad_(True)
    loss = K.cross_entropy(x[..., 2:V + 2], labels.to(DEV), reduction=reduction)
    up = torch.full(loss.shape, 2.0 ** 14, device=DEV)
    if reduction == "none":
        up[0, :2] = 1.0
    for retain in (True, False):
        got = torch.autograd.grad(loss, x, up, retain_graph=retain)[0][..., 2:V + 2].double().cpu()
        p = torch.softmax(wide[..., 2:V + 2].double(), -1)
        hot = torch.zeros_like(p).scatter_(-1, labels.clamp(min=0)[..., None], 1.0)
        f = (up.double().cpu().expand(rows) / (n - 1 if reduction == "mean" else 1) * (labels != -100))[..., None]
        want, size = (p - hot) * f, (p + hot) * f
        # one rounding of the result (two where the kept gradient is scaled, and the smallest numbers of both)
        roundings = 1 if dtype == torch.float16 else 2
        tiny = TINY[dtype] * (1 if dtype == torch.float16 else 2.0 ** 14 + 1)
        bar = roundings * torch.finfo(dtype).eps / 2 * want.abs() + 3 * SUM * size + tiny
        assert bool(((got - want).abs() <= bar).all())


def test_loss_is_the_same_every_time():
    import kvm_amd as K

    x = _logits(300, 5003, torch.bfloat16, 120).to(DEV).requires_grad_(True)
    teacher = K.TopLogits(*(t.to(DEV) if isinstance(t, torch.Tensor) else t
                            for t in _teacher(300, 5003, 50, 121, temperature=2.0)))
    labels = torch.randint(0, 5003, (300,), generator=_gen(122)).to(DEV)
    runs = []
    for _ in range(3):
        loss = K.distillation_loss(x, teacher, labels, label_weight=0.3)
        runs.append((loss.detach(), torch.autograd.grad(loss, x)[0]))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))


def test_loss_refusals_on_the_gpu():
    import kvm_amd as K

    x = torch.zeros(3, 8, device=DEV)
    lab = torch.zeros(3, dtype=torch.long, device=DEV)
    v, i = torch.zeros(3, 2, device=DEV), torch.zeros(3, 2, dtype=torch.long, device=DEV)
    for bad in (lab[:2], lab.float(), lab.cpu()):
        with pytest.raises(ValueError, match="labels"):
            K.cross_entropy(x, bad)
    for teacher, kw, text in (
            (K.TopLogits(v, i[:, :1]), {}, "shape"), (K.TopLogits(v[:2], i[:2]), {}, "shape"),
            (K.TopLogits(v.double(), i), {}, "teacher values"), (K.TopLogits(v, i.float()), {}, "teacher indices"),
            (K.TopLogits(v, i, torch.zeros(2, device=DEV)), {}, "rest"), (K.TopLogits(v, i, None, 0.0), {}, "temperature"),
            (K.TopLogits(v, i), dict(label_weight=0.5), "needs labels"),
            (K.TopLogits(v, i), dict(label_weight=1.5, labels=lab), "label_weight"),
            (K.TopLogits(v.cpu(), i), {}, "device"),
            (K.TopLogits(v[:, :0], i[:, :0]), {}, "values per row")):
        with pytest.raises(ValueError, match=text):
            K.distillation_loss(x, teacher, **kw)


# ---------------------------------------------------------------- streams and graphs

def test_operators_in_a_captured_graph():
    """Sampling, a teacher's scores and a training loss with its backward,
    captured once and replayed on new inputs, eager work between the replays."""
    import kvm_amd as K

    n, V, k = 33, 3001, 24
    x = _logits(n, V, torch.bfloat16, 130).to(DEV).requires_grad_(True)
    tx = _logits(n, V, torch.bfloat16, 131).to(DEV)
    u = torch.rand(n, generator=_gen(132)).to(DEV)
    labels = torch.randint(0, V, (n,), generator=_gen(133)).to(DEV)

    def step():
        tok, lp = K.sample_tokens(x.detach(), u, temperature=0.9, top_p=0.9, return_logprobs=True)
        teacher = K.top_logits(tx, k, temperature=2.0)
        loss = K.distillation_loss(x, teacher, labels, label_weight=0.25)
        return tok, lp, teacher.values, teacher.indices, teacher.rest, loss.detach(), torch.autograd.grad(0.5 * loss, x)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for r in range(4):
        with torch.no_grad():
            x.copy_(_logits(n, V, torch.bfloat16, 140 + r))
            tx.copy_(_logits(n, V, torch.bfloat16, 150 + r))
            u.copy_(torch.rand(n, generator=_gen(160 + r)))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step())), f"replay {r}"
    graph.reset()


def test_loss_and_gradient_captured_apart():
    """A backward replayed on an eager loss gives the same gradient every time,
    and an eager backward of a replayed loss one that later replays leave alone."""
    import kvm_amd as K

    x = _logits(17, 1003, torch.float32, 180).to(DEV).requires_grad_(True)
    labels = torch.randint(0, 1003, (17,), generator=_gen(181)).to(DEV)
    up = torch.tensor(0.5, device=DEV)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()

    def expected():
        return torch.autograd.grad(K.cross_entropy(x, labels), x, up)[0]

    with torch.cuda.stream(side):
        want = expected()
        loss = K.cross_entropy(x, labels)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        grad, = torch.autograd.grad(loss, x, up, retain_graph=True)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, want)
        grad.zero_()
    graph.reset()

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        loss = K.cross_entropy(x, labels)
    kept = []
    for i in range(3):
        x.data.copy_(_logits(17, 1003, torch.float32, 182 + i))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        kept.append((torch.autograd.grad(loss, x, up, retain_graph=True)[0], expected()))
    torch.cuda.synchronize()
    assert all(torch.equal(got, want) for got, want in kept)
    del loss
    graph.reset()


def test_operators_on_two_streams():
    import kvm_amd as K

    streams = [torch.cuda.Stream() for _ in range(2)]
    x = [_logits(64, 20011, torch.bfloat16, 170 + i).to(DEV).requires_grad_(True) for i in range(2)]
    labels = torch.randint(0, 20011, (64,), generator=_gen(172)).to(DEV)
    u = torch.rand(64, generator=_gen(173)).to(DEV)
    torch.cuda.synchronize()

    def work(t):
        loss = K.cross_entropy(t, labels)
        return torch.autograd.grad(loss, t)[0], K.sample_tokens(t.detach(), u, top_p=0.9), K.top_logits(t.detach(), 9).indices

    got = [[], []]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = work(x[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[i], work(x[i])))


# ---------------------------------------------------------------- the decoder

def _model(seed, softcap=0.0):
    from kvm_amd.backbone import MixerConfig, RWKV7BackboneForCausalLM, init_random_

    cfg = MixerConfig(vocab_size=515, num_hidden_layers=2, num_attention_heads=4, hidden_size=256,
                      mup_base_dim=256, use_tokenshift_att=1, use_tokenshift_ffn=1, residual_scale=0.5,
                      rope_partial_dim=32, chunk_len=64, n_bswa_chunks=2, state_min_len=64,
                      state_budget_mode="fixed", sink_len=1, logit_softcap=softcap)
    with torch.device("meta"):
        model = RWKV7BackboneForCausalLM(cfg)
    return init_random_(model.to_empty(device=DEV).to(torch.bfloat16), seed)


def test_decoder_samples_eagerly_and_from_a_graph():
    from kvm_amd import DecodeGraph, StatesDictCache, sample_tokens

    model = _model(1).eval()
    ids = torch.randint(0, 515, (3, 200), generator=_gen(200)).to(DEV)
    n = 40
    u = torch.rand(3, n, generator=_gen(201)).to(DEV)
    kw = dict(temperature=torch.tensor([0.0, 0.8, 1.2], device=DEV), top_k=50, top_p=0.95, uniforms=u)
    tokens, lp = model.generate_sampled(ids, n, **kw, return_logprobs=True)
    runner = DecodeGraph(model, StatesDictCache())
    tokens_g, lp_g = runner.generate_sampled(ids, n, **kw, return_logprobs=True)
    runner.close()
    assert torch.equal(tokens, tokens_g) and torch.equal(lp, lp_g)
    assert torch.equal(tokens[:1], model.generate_greedy(ids, n)[:1])
    # each token is the one that the logits before it give
    seen = torch.cat([ids, tokens], 1)
    cache = StatesDictCache()
    with torch.no_grad():
        logits = model(input_ids=ids, past_key_values=cache, use_cache=True,
                       cache_position=torch.arange(200, device=DEV), logits_to_keep=1).logits[:, -1]
        for s in range(n):
            assert torch.equal(sample_tokens(logits, u[:, s], temperature=kw["temperature"], top_k=50, top_p=0.95),
                               tokens[:, s])
            logits = model(input_ids=seen[:, 200 + s:201 + s], past_key_values=cache, use_cache=True,
                           cache_position=torch.tensor([200 + s]), logits_to_keep=1).logits[:, -1]
    a = model.generate_sampled(ids, 5, generator=torch.Generator(device=DEV).manual_seed(3))
    b = model.generate_sampled(ids, 5, generator=torch.Generator(device=DEV).manual_seed(3))
    assert torch.equal(a, b) and a.shape == (3, 5)


@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_on_policy_distillation_step(softcap):
    """Sample a rollout from the student, score it with a teacher, train the
    student on it: the loss and its gradient at the LM head against torch in
    64 bits from the same hidden states, and an update that uses it."""
    student, teacher = _model(2, softcap).train(), _model(3, softcap).eval()
    prompt = torch.randint(0, 515, (2, 100), generator=_gen(210)).to(DEV)
    rollout = student.generate_sampled(prompt, 29, top_p=0.9, generator=torch.Generator(device=DEV).manual_seed(1))
    assert student.training and all(m.training for m in student.modules())
    again = _model(2, softcap).eval().generate_sampled(prompt, 29, top_p=0.9,
                                                       generator=torch.Generator(device=DEV).manual_seed(1))
    assert torch.equal(rollout, again)  # a model in training samples as it does in evaluation
    ids = torch.cat([prompt, rollout], 1)
    labels = ids.clone()
    labels[:, :100] = -100                         # the prompt is not learnt
    scores = teacher.top_logits(ids, 16, temperature=2.0)
    assert scores.values.shape == (2, 129, 16)
    loss = student.loss(ids, labels, teacher=scores, label_weight=0.5)
    loss.backward()
    with torch.no_grad():
        full = teacher(input_ids=ids).logits
        assert torch.equal(scores.values, full.gather(-1, scores.indices).bfloat16())
    hidden = student.transformer(input_ids=ids).last_hidden_state.detach()
    w = student.lm_head.weight.detach().clone().requires_grad_(True)
    logits = torch.nn.functional.linear(hidden, w)
    if softcap:
        logits = softcap * torch.tanh(logits / softcap)
    targets = torch.cat([labels[:, 1:], torch.full((2, 1), -100, device=DEV)], 1).view(-1).cpu()
    want, grad, _, counted = O.loss_rows(logits.detach().view(-1, 515).cpu(), targets,
                                         tuple(t.cpu().flatten(0, 1) if isinstance(t, torch.Tensor) else t
                                               for t in scores), 0.5)
    count = int(counted.sum())
    assert count == 2 * 29
    assert abs(float(loss.detach()) - float(want.sum()) / count) <= 12 * SUM + abs(float(want.sum())) / count * 2.0 ** -22
    logits.backward((grad / count).view_as(logits).to(DEV, torch.bfloat16))
    # The same rounded gradient but for values next to a rounding border (half
    # a step of 2^-8 each), through the same products.
    diff = (student.lm_head.weight.grad.double() - w.grad.double()).norm()
    assert float(diff) <= 2.0 ** -8 * float(w.grad.double().norm())
    before = [p.detach().clone() for p in student.parameters()]
    torch.optim.SGD(student.parameters(), lr=0.5).step()
    assert sum(not torch.equal(a, b) for a, b in zip(before, student.parameters())) > len(before) // 2
    hard = student.loss(ids, labels)
    assert hard.dim() == 0 and hard.requires_grad
    assert student.loss(ids, labels, reduction="none").shape == ids.shape
