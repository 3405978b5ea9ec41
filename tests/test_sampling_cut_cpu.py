"""Where top-p's share of a row ends, estimated from a histogram: every CTA of a
cluster, and every thread that looks, has to find one and the same bin.

The kernel's block scan (16 warps of 32 threads, four bins a thread) restated in
numpy.  Running sums in fp32 overlap by their rounding, so two threads can both
hold the share's end; sums of whole numbers cannot.
"""
import numpy as np
import pytest

F32 = np.float32
BINS, WARPS, LANES, PER = 2048, 16, 32, 4


def _steps(x):
    """Inclusive running sums along the last axis, in the order of the shuffles."""
    off = 1
    while off < x.shape[-1]:
        y = x.copy()
        y[..., off:] += x[..., :-off]
        x, off = y, 2 * off
    return x


def _intervals(m):
    """Start and end of each bin's share, m [BINS] in the scan's own number type."""
    m = m.reshape(WARPS * LANES, PER)
    own = m[:, 0]
    for i in range(1, PER):
        own = own + m[:, i]
    own = own.reshape(WARPS, LANES)
    inc = _steps(own)
    warps = _steps(inc[:, -1].copy())
    at = ((warps - inc[:, -1])[:, None] + inc - own).reshape(-1)
    lo, hi = [], []
    for i in range(PER):
        lo.append(at)
        at = at + m[:, i]
        hi.append(at)
    return np.stack(lo, 1).reshape(-1), np.stack(hi, 1).reshape(-1), warps[-1]


def row_and_shares(seed, most):
    """A row of logits and shares that end where two fp32 intervals overlap."""
    logits = np.random.default_rng(seed).standard_normal(151936).astype(F32) * F32(2.5)
    top = logits.max()
    scale = F32(BINS - 1) / F32(min(top - logits.min(), F32(64)))
    counts = np.bincount(np.minimum(BINS - 1, ((top - logits) * scale).astype(int)), minlength=BINS)
    e = np.exp(-(np.arange(BINS, dtype=F32) + F32(0.5)) / scale, dtype=F32)
    m = counts.astype(F32) * (e + F32(1e-30))
    lo, hi, whole = _intervals(m)
    shares = []
    for i in range(BINS - 1):
        if m[i] > 0 and m[i + 1] > 0 and hi[i] > lo[i + 1]:
            p = F32(np.nextafter(lo[i + 1], F32(np.inf)) / whole)
            owners = np.flatnonzero((m > 0) & (lo < p * whole) & (hi >= p * whole))
            if len(owners) > 1:
                shares.append((float(p), owners))
    return logits, counts, e, shares[:most]


@pytest.mark.parametrize("seed", [0, 1, 2])
def test_whole_numbers_have_one_owner(seed):
    _, counts, e, shares = row_and_shares(seed, 64)
    assert shares   # fp32 sums do overlap here
    m = counts.astype(np.uint64) * ((e * F32(2.0 ** 40)).astype(np.uint64) + np.uint64(1))
    lo, hi, whole = _intervals(m)
    assert lo[0] == 0 and (hi[:-1] == lo[1:]).all() and hi[-1] == whole == m.sum()
    for p, owners in shares:
        want = np.uint64(max(1, min(int(whole), int(np.ceil(np.float64(F32(p)) * float(whole))))))
        one = np.flatnonzero((lo < want) & (hi >= want))
        assert len(one) == 1 and abs(int(one[0]) - int(owners[0])) <= 2
