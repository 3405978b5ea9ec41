"""Sampling on the GPU against the float64 oracle, row by row: tokens are equal.

The kernel's weights have a relative error below 1e-13 and steps of 2^-44, the
oracle's below 1e-15; a token could differ only where u times the sum lies that
near to a running sum, which the fixed inputs here do not hit (probability below
1e-6 for all rows together).  Log probabilities are rounded to fp32 once (half a
step, 2^-24) from values good to 1e-12.
"""
import numpy as np
import pytest
import torch

from helm_b200 import _capi
from oracle import serving

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("CUDA device required")
    return torch.device("cuda:0")


def _check(dev, logits, u, temp=None, top_k=None, top_p=None, min_p=None, want_logp=True):
    b = logits.shape[0]
    f = lambda x, dt: None if x is None else torch.tensor(x, dtype=dt, device=dev)  # noqa: E731
    args = dict(temperature=f(temp, torch.float32), top_k=f(top_k, torch.int32),
                top_p=f(top_p, torch.float32), min_p=f(min_p, torch.float32))
    ut = f(u, torch.float32)
    logp = torch.empty(b, device=dev) if want_logp else None
    ids = _capi.sample_tokens(logits, ut, logprobs=logp, **args)
    rows = logits.double().cpu().numpy()
    get = lambda name, i, d: d if args[name] is None else float(args[name][i])  # noqa: E731
    for i in range(b):
        tok, lp = serving.sample(rows[i], float(ut[i]), get("temperature", i, 1.0),
                                 int(get("top_k", i, 0)), get("top_p", i, 1.0), get("min_p", i, 0.0))
        assert int(ids[i]) == tok, (i, int(ids[i]), tok)
        if want_logp:
            got = float(logp[i])
            assert got == lp or abs(got - lp) <= abs(lp) * 2.0 ** -24 * 1.01 + 1e-11, (i, got, lp)
    return ids


def _logits(b, v, seed, dtype, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, v, generator=g) * spread
    x[:, ::max(1, v // 20)] += 6 * torch.rand(b, len(range(0, v, max(1, v // 20))), generator=g)
    return x.to(dtype), torch.rand(b, generator=g).tolist()


@pytest.mark.parametrize("v", [1, 2, 31, 33, 1000, 4097, 32000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_filters(dev, v, dtype):
    b = 12
    x, u = _logits(b, v, v, dtype)
    x = x.to(dev)
    i = np.arange(b)
    temp = np.where(i % 6 == 5, 0.0, 0.5 + i / 10)
    k = np.where(i % 3 == 0, 0, 1 + i * 5)
    p = np.where(i % 4 == 1, 1.0, 0.3 + i / 20)
    m = np.where(i % 2 == 0, 0.0, 0.02 * i)
    _check(dev, x, u)
    _check(dev, x, u, temp=temp)
    _check(dev, x, u, temp=temp, top_k=k)
    _check(dev, x, u, temp=temp, top_p=p)
    _check(dev, x, u, min_p=m)
    _check(dev, x, u, temp=temp, top_k=k, top_p=p, min_p=m)
    _check(dev, x, u, temp=temp, top_k=k, top_p=p, min_p=m, want_logp=False)


@pytest.mark.parametrize("b,v,dtype", [(1, 151936, torch.bfloat16), (3, 151936, torch.float32),
                                       (1, 262144, torch.float32), (160, 50001, torch.float16)])
def test_large_vocabularies(dev, b, v, dtype):
    x, u = _logits(b, v, b + v, dtype)
    i = np.arange(b)
    _check(dev, x.to(dev), u, temp=0.7 + 0.01 * (i % 40), top_p=np.full(b, 0.95),
           top_k=np.where(i % 2, 0, 50))
    _check(dev, x.to(dev), u)


def test_unaligned_and_strided_rows(dev):
    x, u = _logits(5, 1003, 3, torch.bfloat16)
    wide = torch.full((5, 1011), 99.0, dtype=torch.bfloat16, device=dev)
    wide[:, 3:1006] = x.to(dev)
    _check(dev, wide[:, 3:1006], u, top_p=[0.9] * 5)


def test_equal_logits(dev):
    """One bin holds everything: thresholds by index, bisected; running sums are whole numbers."""
    x = torch.zeros(8, 5000, device=dev)
    u = [0.0, 0.25, 0.5, 0.75, 0.9, 0.999, 0.1, 0.33]
    _check(dev, x, u)
    _check(dev, x, u, top_k=[1, 7, 1024, 1025, 4999, 5000, 0, 2000])
    _check(dev, x, u, top_p=[0.0, 0.001, 0.25, 0.5, 0.75, 0.999, 1.0, 0.125])
    _check(dev, x, u, top_k=[4000] * 8, top_p=[0.5] * 8, min_p=[1.0] * 8)
    ids = _check(dev, x, u, temp=[0.0] * 8)
    assert (ids == 0).all()


def test_ties_at_the_border(dev):
    """Values on a coarse grid: many candidates share the threshold's logit."""
    g = torch.Generator().manual_seed(5)
    x = torch.randint(-4, 3, (10, 6000), generator=g).float().to(dev)
    u = torch.rand(10, generator=g).tolist()
    _check(dev, x, u, top_k=[1, 5, 100, 857, 858, 1500, 3000, 5999, 2, 3])
    _check(dev, x, u, top_p=[0.05, 0.1, 0.3, 0.5, 0.6, 0.7, 0.8, 0.9, 0.95, 0.99])
    _check(dev, x, u, min_p=[float(np.float32(np.exp(-1.5)))] * 10)


def test_masked_outlying_and_non_finite_logits(dev):
    inf, nan = float("inf"), float("nan")
    x, u = _logits(10, 3000 + 9, 7, torch.float32)
    x[0, 1:] = -inf                          # one candidate
    x[1] = -inf                              # none
    x[2] = nan                               # none
    x[3, ::2] = nan
    x[4, 100:] = -inf
    x[5, :2000] = torch.finfo(torch.float32).min
    x[6, 17] = 1e4                           # far above the rest
    x[7, 5] = x[7, 700] = inf                # infinities share the weight
    x[8, ::3] = -1e30
    x[9] = -inf
    x[9, 2500] = -3e38
    k = [5, 5, 5, 900, 200, 1500, 3, 1, 2500, 7]
    p = [0.9, 0.9, 0.9, 0.8, 0.99, 0.7, 0.5, 0.3, 0.99, 0.5]
    ids = _check(dev, x.to(dev), u)
    assert ids[1] == ids[2] == -1
    _check(dev, x.to(dev), u, top_k=k)
    _check(dev, x.to(dev), u, top_p=p)
    _check(dev, x.to(dev), u, top_k=k, top_p=p, temp=[0.3, 1, 1, 5, 0.01, 1, 100, 1, 0.7, 1])
    _check(dev, x.to(dev), u, temp=[0.0] * 10)


def test_border_values_of_the_parameters(dev):
    x, _ = _logits(8, 500, 9, torch.float32)
    u = [0.0, float(np.nextafter(np.float32(1), np.float32(0))), 1.0, 2.0, 0.5, 0.5, 0.5, 0.5]
    ids = _check(dev, x.to(dev), u[:2] + [0.999999] * 2 + u[4:], top_k=[-3, 0, 500, 501, 1, 499, 2, 3])
    # u of one and above draws the last candidate that is left
    got = _capi.sample_tokens(x.to(dev), torch.tensor(u, device=dev))
    assert (got[2:4] == 499).all()
    nan = torch.full((8,), float("nan"), device=dev)
    greedy = _capi.sample_tokens(x.to(dev), torch.tensor(u, device=dev), temperature=nan)
    assert torch.equal(greedy.cpu(), x.argmax(1))
    assert ids.dtype == torch.int64


def test_result_does_not_depend_on_the_launch(dev):
    """The same row alone (many CTAs) and in a large batch (few CTAs a row): the same token."""
    x, _ = _logits(1, 70000, 11, torch.bfloat16)
    x = x.to(dev)
    u = torch.rand(200, device=dev)
    p = torch.full((200,), 0.9, device=dev)
    many = _capi.sample_tokens(x.expand(200, -1), u, top_p=p)
    one = torch.cat([_capi.sample_tokens(x, u[i:i + 1], top_p=p[i:i + 1]) for i in range(200)])
    assert torch.equal(many, one)


def test_captured_and_replayed(dev):
    x, u = _logits(4, 32000, 13, torch.bfloat16)
    logits, ut = x.to(dev), torch.tensor(u, device=dev)
    out = torch.empty(4, dtype=torch.int64, device=dev)
    p = torch.full((4,), 0.8, device=dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _capi.sample_tokens(logits, ut, top_p=p, out=out)
    for seed in range(3):
        x, u = _logits(4, 32000, 17 + seed, torch.bfloat16)
        logits.copy_(x)
        ut.copy_(torch.tensor(u))
        g.replay()
        torch.cuda.synchronize(dev)
        for i in range(4):
            assert int(out[i]) == serving.sample(x[i].double().numpy(), float(np.float32(u[i])),
                                                 top_p=float(np.float32(0.8)))[0]


def test_border_of_the_sorted_list(dev):
    """Exactly as many candidates up to the k-th one's bin as are sorted in one go, and more of
    them within rounding of that bin's edge: they do not fit, and the row takes the long way."""
    v = 3000
    x = torch.full((2, v), -60.0)
    x[:, 0] = 10.0
    x[:, 1:1024] = 10.0 - 0.6
    edge = 20 / (2047 / 64)   # the bins are 64 / 2047 wide; 0.6 lies in the 20th
    x[:, 1024:1080] = float(np.float32(10.0 - edge * (1 + 5e-6)))
    u = [0.3, 0.9]
    _check(dev, x.to(dev), u, top_k=[1024, 1024])
    _check(dev, x.to(dev), u, top_k=[1024, 1050], top_p=[0.9, 0.99])


def test_few_heavy_candidates_with_gaps(dev):
    """Top-p's share ends next to a gap of many empty bins: the estimate may fall on either side."""
    x = torch.full((40, 5000), -20.0)
    x[:, ::50] = 6.0 - 0.21 * torch.arange(100)
    l = x.double().numpy()
    w = np.sort(np.exp(l[0] - l[0].max()))[::-1].cumsum() / np.exp(l[0] - l[0].max()).sum()
    # shares just below and above the running sums of the first candidates
    p = [float(np.float32(w[i // 2] * (1 + (1e-3 if i % 2 else -1e-3)))) for i in range(40)]
    g = torch.Generator().manual_seed(3)
    _check(dev, x.to(dev), torch.rand(40, generator=g).tolist(), top_p=[min(q, 0.9999) for q in p])


def test_infinities_and_a_large_k(dev):
    """k reaches far beyond the infinite logits, into the last bin of all."""
    x, u = _logits(4, 30000, 9, torch.float32)
    x[0, 5::1000] = float("inf")
    x[1, 100] = float("inf")
    x[2, ::2] = float("inf")
    k = [5000, 20000, 20000, 5000]
    _check(dev, x.to(dev), u, top_k=k)
    _check(dev, x.to(dev), u, top_k=k, top_p=[0.5, 0.9, 0.999, 0.9], temp=[1.0, 2.0, 0.1, 50.0])


def test_long_bf16_rows_of_every_kind(dev):
    """As many rows as SMs: weights come from the table of bf16 values, whatever the row holds."""
    b, v = 160, 65544
    x, u = _logits(b, v, v, torch.bfloat16)
    for i in range(b):
        row, kind = x[i], i % 10
        if kind == 1:
            row[::3] = float("-inf")
        elif kind == 2:
            row[::2] = 0.0
            row[1::8] = -0.0
        elif kind == 3:
            row *= 2.0 ** -20                 # all weights nearly alike
        elif kind == 4:
            row -= 300                        # all negative, coarse steps
        elif kind == 5:
            row *= 1e4
            row[7] = float("nan")
        elif kind == 6:
            row[5::1000] = float("inf")
        elif kind == 7:
            row[:] = row[0]
        elif kind == 8:
            row[:-3] = float("-inf")
            row[-2] = torch.finfo(torch.bfloat16).min
        elif kind == 9:
            row[::5] *= 1e-30                 # far below the table's magnitudes
    x = x.to(dev)
    i = np.arange(b)
    temp = np.where(i % 7 == 6, 0.0, np.where(i % 20 == 15, 3e4, 0.4 + i / 100))
    p = np.where(i % 3 == 1, 0.2 + i / 250, 1.0)
    k = np.where(i % 4 == 2, 1 + 37 * i, 0)
    m = np.where(i % 5 == 3, 0.01, 0.0)
    _check(dev, x, u, temp=temp, top_k=k, top_p=p, min_p=m)
    _check(dev, x, u, temp=temp, top_p=p, want_logp=False)


def test_long_bf16_rows_cut_at_every_place(dev):
    """Filters that end among values far below the largest, at zeros of both signs, at
    the last candidate, among candidates without weight, and within many equal ones."""
    b, v = 160, 65536
    x, u = _logits(b, v, 77, torch.bfloat16)
    g = torch.Generator().manual_seed(78)
    for i in range(b):
        row, kind = x[i], i % 5
        if kind == 1:
            row *= 1e-30
            row[i] = 2.0
        elif kind == 2:
            row[torch.randperm(v, generator=g)[:50000]] = 0.0
            row[::7] = -0.0
            row.clamp_(max=0.0)
        elif kind == 3:
            row[:] = torch.randint(0, 3, (v,), generator=g).to(torch.bfloat16)
        elif kind == 4:
            row[100:] -= 1000
            row[v // 2:] = float("-inf")
    x = x.to(dev)
    i = np.arange(b)
    p = 0.03 + 0.96 * (i * 37 % b) / b
    k = np.where(i % 3 == 0, 1 + i * 400, np.where(i % 3 == 1, v - 1 - i, 0))
    _check(dev, x, u, top_p=p)
    _check(dev, x, u, top_k=k, top_p=np.where(i % 4 == 1, p, 1.0))


def test_wrapper_refusals(dev):
    x, u = torch.zeros(2, 8, device=dev), torch.zeros(2, device=dev)
    for bad in (lambda: _capi.sample_tokens(x.t(), u), lambda: _capi.sample_tokens(x, u[:1]),
                lambda: _capi.sample_tokens(x, u.double()), lambda: _capi.sample_tokens(x.int(), u),
                lambda: _capi.sample_tokens(x, u, top_k=u),
                lambda: _capi.sample_tokens(x, u, temperature=u.cpu()),
                lambda: _capi.sample_tokens(x[0], u)):
        with pytest.raises(_capi.HelmError):
            bad()
