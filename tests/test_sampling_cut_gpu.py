"""Sampling where a filter's end is hard to place (GPU), token for token against the
float64 oracle; tolerances as in test_sample_tokens_gpu.py."""
import numpy as np
import pytest
import torch

from helm_b200 import _capi
from test_sample_tokens_gpu import _check, dev  # noqa: F401
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


def test_no_rows(dev):  # noqa: F811
    x, u = torch.empty(0, 100, device=dev), torch.empty(0, device=dev)
    ids = _capi.sample_tokens(x, u, logprobs=torch.empty(0, device=dev))
    assert ids.shape == (0,) and ids.dtype == torch.int64
