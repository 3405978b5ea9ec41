"""Decode attention over 4-bit pages where keys differ by many orders of magnitude in
weight, and where a visible score is NaN (GPU, against the float64 oracle).

P is held in fp16 with its largest value between 2^11 and 2^15, so a weight is off by
half a step: 2^-11 of itself, or 2^-25 / 2^11 = 2^-36 of the largest one (the second
part is what `tiny` adds up over the keys).
"""
import numpy as np
import pytest
import torch

from helm_b200 import _capi
from oracle import fp4

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("CUDA device required")
    return torch.device("cuda:0")


def _pool(dev, k, v, page):
    """A pool that holds k, v [T, Hkv, D] (exact in 4 bits) in order, and its table."""
    n, hkv, d = k.shape
    pages = -(-n // page)
    pool = _capi.fp4_pool(pages, hkv, page, d, dev)
    _capi.kv_append_fp4(k=k.to(dev), v=v.to(dev), pool=pool, slot_rows=torch.arange(n, device=dev),
                        page_size=page)
    table = torch.arange(pages, dtype=torch.int32, device=dev).view(1, -1)
    return pool, table, torch.tensor([n], dtype=torch.int32, device=dev)


@pytest.mark.parametrize("nats", [15.0, 17.5, 20.0])
@pytest.mark.parametrize("dtype,hq", [(BF16, 4), (FP16, 4), (FP16, 6), (BF16, 12)])
def test_many_light_keys_beside_a_heavy_one(dev, dtype, hq, nats):
    """One key with V = 0 takes nearly all of the weight: O is what the others leave.  With a
    hint of 32 tokens one warp meets all of the keys, against one running maximum."""
    n, d, page, heavy = 131072, 64, 64, 17
    g = np.random.default_rng(int(nats))
    levels = np.concatenate([fp4.E2M1, -fp4.E2M1])
    v = levels[g.integers(0, 16, (997, d))]
    v[:, ::16] = 6.0          # every block's scale is 1
    v = np.tile(v, (n // 997 + 1, 1))[:n]
    v[heavy] = 0
    k = np.zeros((n, d))
    k[heavy, 0] = 6.0
    q = torch.zeros(1, hq, d)
    q[:, :, 0] = 1.0
    scale = float(np.float32(nats / 6))
    pool, table, lens = _pool(dev, torch.from_numpy(k[:, None]).to(dtype),
                              torch.from_numpy(v[:, None]).to(dtype), page)
    lse = torch.empty(1, hq, device=dev)
    kw = dict(num_kv_heads=1, page_size=page, scale=scale)
    for mask, hint in ((None, 0), (None, 32), (torch.zeros(1, n, device=dev), 32)):
        out, _ = _capi.paged_decode_attention_fp4(q.to(dtype).to(dev), pool, table, lens, lse=lse,
                                                  mask=mask, max_kv_len_hint=hint, **kw)
        w = np.full(n, np.exp(-6 * scale))
        w[heavy] = 1
        want, size = w @ v / w.sum(), w @ np.abs(v) / w.sum()
        half = torch.finfo(dtype).eps / 2
        tiny = n * 2.0 ** -36 * 6
        # l: each of eight lanes adds up four of the 32 keys of a unit, two at a time, in
        # fp32: n / 16 additions to a sum of at most l, each off by 2^-24 of it at most
        l_err = n / 16 * 2.0 ** -24
        # scores are exact up to one rounding, exp2 and the other sums below 2^-20 of their size
        tol = (size * (2.0 ** -11 + 2.0 ** -20 + l_err) + np.abs(want) * half * 1.001 + tiny
               + 2.0 ** -25)
        got = out.double().cpu().numpy()[0]
        assert (np.abs(got - want) <= tol).all(), np.abs((got - want) / tol).max()
        off = lse.double().cpu().numpy() - (6 * scale + np.log(w.sum()))
        assert (np.abs(off) <= l_err + 20 * 2.0 ** -22).all(), np.abs(off).max()


@pytest.mark.parametrize("dtype,hq,d", [(BF16, 8, 128), (FP16, 4, 64), (BF16, 4, 256), (FP16, 24, 128)])
def test_a_visible_nan_is_not_hidden_by_the_soft_cap(dev, dtype, hq, d):
    g = torch.Generator().manual_seed(d + hq)
    n, hkv, page = 90, 2, 16
    k = torch.randn(n, hkv, d, generator=g).to(dtype)
    v = torch.randn(n, hkv, d, generator=g).to(dtype)
    q = torch.randn(1, hq, d, generator=g).to(dtype)
    kw = dict(num_kv_heads=hkv, page_size=page, scale=0.1)

    def run(k, q, cap):
        pool, table, lens = _pool(dev, k, v, page)
        lse = torch.empty(1, hq, device=dev)
        out, _ = _capi.paged_decode_attention_fp4(q.to(dev), pool, table, lens, lse=lse, softcap=cap,
                                                  **kw)
        return out.cpu()[0], lse.cpu()[0]

    for cap in (0.0, 30.0):
        ref, ref_lse = run(k, q, cap)
        bad_k = k.clone()
        bad_k[37, 1, 5] = float("nan")       # its block of KV head 1
        out, lse = run(bad_k, q, cap)
        clean = slice(0, hq // 2)
        assert torch.equal(out[clean], ref[clean]) and torch.equal(lse[clean], ref_lse[clean])
        assert torch.isnan(out[hq // 2:]).all() and torch.isnan(lse[hq // 2:]).all()
        bad_q = q.clone()
        bad_q[0, 1, 3] = float("nan")
        out, lse = run(k, bad_q, cap)
        others = [h for h in range(hq) if h != 1]
        assert torch.equal(out[others], ref[others]) and torch.equal(lse[others], ref_lse[others])
        assert torch.isnan(out[1]).all() and torch.isnan(lse[1]).all()
