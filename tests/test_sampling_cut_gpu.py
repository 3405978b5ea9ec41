"""Sampling where a filter's end is hard to place (GPU), token for token against the
float64 oracle; tolerances as in test_sample_tokens_gpu.py."""
import numpy as np
import pytest
import torch

from helm_b200 import _capi
from test_sample_tokens_gpu import _check, _logits, dev  # noqa: F401
from test_sampling_cut_cpu import row_and_shares

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", [0, 1])
def test_shares_that_end_on_a_border_of_fp32_sums(dev, seed):  # noqa: F811
    """Rows held by a cluster of eight CTAs: all of them use the same bins."""
    logits, _, _, shares = row_and_shares(seed, 16)
    p = [s[0] for s in shares]
    x = torch.from_numpy(logits).to(dev).expand(len(p), -1)
    u = torch.rand(len(p), generator=torch.Generator().manual_seed(seed)).tolist()
    _check(dev, x, u, top_p=p)
    _check(dev, x, u, top_p=p, top_k=np.where(np.arange(len(p)) % 2, 0, 150000))
    assert _capi.device_status(dev) == 0


@pytest.mark.parametrize("dtype,v", [(torch.float32, 8204), (torch.float32, 40000),
                                     (torch.float16, 8200), (torch.float16, 40000),
                                     (torch.bfloat16, 8200), (torch.bfloat16, 65528)])
def test_whole_rows_of_a_large_batch(dev, dtype, v):  # noqa: F811
    """As many rows as SMs, each a whole number of vectors: one CTA a row, no table of values."""
    b = 160
    x, u = _logits(b, v, v, dtype)
    g = torch.Generator().manual_seed(v)
    for i in range(b):
        row, kind = x[i], i % 8
        if kind == 1:
            row[::3] = float("-inf")
        elif kind == 2:
            row[:] = torch.randint(-3, 3, (v,), generator=g).to(dtype)   # many equal logits
        elif kind == 3:
            row[7::97] = float("nan")
        elif kind == 4:
            row[5::1000] = float("inf")
        elif kind == 5:
            row[:] = row[0]
        elif kind == 6:
            row *= 2.0 ** -12                 # all weights nearly alike
        elif kind == 7:
            row[:-3] = float("-inf")
    x = x.to(dev)
    i = np.arange(b)
    temp = np.where(i % 7 == 6, 0.0, 0.4 + i / 100)
    p = np.where(i % 3 == 1, 0.2 + i / 250, 1.0)
    k = np.where(i % 4 == 2, 1 + 37 * i, np.where(i % 4 == 3, 1 + i % 60, 0))
    m = np.where(i % 5 == 3, 0.01, 0.0)
    _check(dev, x, u)
    _check(dev, x, u, temp=temp, top_k=k, top_p=p, min_p=m)
    _check(dev, x, u, temp=temp, top_p=0.03 + 0.96 * (i * 37 % b) / b, want_logp=False)
    _check(dev, x, u, top_k=1 + i * 37 % (v - 1), want_logp=False)
    assert _capi.device_status(dev) == 0


def test_no_rows(dev):  # noqa: F811
    x, u = torch.empty(0, 100, device=dev), torch.empty(0, device=dev)
    ids = _capi.sample_tokens(x, u, logprobs=torch.empty(0, device=dev))
    assert ids.shape == (0,) and ids.dtype == torch.int64
