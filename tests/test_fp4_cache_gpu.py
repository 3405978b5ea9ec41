"""4-bit pages on the GPU: the quantising append, the read-back and the decode
attention, through the C ABI, against the float64 oracle (oracle/fp4.py).

Tolerances.  Append without norm and rotation sees exact inputs: the pool's
bytes are the oracle's.  With them, fp32 rounds every product and sum (64-term
tree and a handful of steps: relative error below 2e-5 of the terms' size), so
a value may fall on the other side of a border only if it lies that near to it:
everything else is equal.  Attention: P is rounded to fp16 (half a step, 2^-11),
scores carry the fp32 error of a D-term product, the output rounds once; the
bound is written out in _check_attention.
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


def _np(t):
    return t.double().cpu().numpy()


# --------------------------------------------------------------------- append --
@pytest.mark.parametrize("d,hkv,page,dtype", [(64, 3, 16, BF16), (128, 2, 48, FP16),
                                              (128, 8, 16, BF16), (256, 1, 32, BF16),
                                              (256, 5, 16, FP16)])
def test_plain_append_writes_the_oracles_bytes(dev, d, hkv, page, dtype):
    g = torch.Generator().manual_seed(d + hkv)
    n, pages = 37, 6
    k = torch.randn(n, hkv, d, generator=g).to(dtype)
    v = torch.randn(n, hkv, d, generator=g).to(dtype) * 3
    k[0] = 0
    k[1, 0, :16] = torch.tensor([6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5] * 2).to(dtype)  # ties
    k[1, 0, 16:32] = -k[1, 0, :16]
    k[2] *= 2.0 ** -9  # subnormal scales
    v[3, 0, 5] = float("inf")
    v[3, 0, 6] = float("-inf")
    v[4, 0, 20] = -0.0
    v[5] = torch.finfo(dtype).max
    rows = torch.randperm(pages * page, generator=g)[:n]
    rows[7] = -1
    pool = torch.full((pages, hkv, page // 16, 18 * d), 0xAB, dtype=torch.uint8)
    want = pool.numpy().copy()
    fp4.write_rows(want, rows.tolist(), _np(k), _np(v), page)
    pool = pool.to(dev)
    _capi.kv_append_fp4(k=k.to(dev), v=v.to(dev), pool=pool, slot_rows=rows.to(dev),
                        page_size=page)
    assert np.array_equal(pool.cpu().numpy(), want)
    kd, vd = _capi.gather_kv_rows_fp4(pool, rows.to(dev), page_size=page, dtype=dtype)
    kw, vw = fp4.read_rows(want, rows.tolist(), page)
    assert np.array_equal(_np(kd), kw) and np.array_equal(_np(vd), vw)
    assert _capi.device_status(dev) == 0


def test_nan_marks_its_block_and_no_other(dev):
    d = 64
    k = torch.ones(1, 1, d, dtype=BF16, device=dev)
    v = torch.ones(1, 1, d, dtype=BF16, device=dev)
    k[0, 0, 17] = float("nan")
    pool = _capi.fp4_pool(1, 1, 16, d, dev)
    rows = torch.tensor([3], device=dev)
    _capi.kv_append_fp4(k=k, v=v, pool=pool, slot_rows=rows, page_size=16)
    kd, vd = _capi.gather_kv_rows_fp4(pool, rows, page_size=16, dtype=BF16)
    nan = torch.isnan(kd[0, 0]).cpu()
    assert nan[16:32].all() and not nan[:16].any() and not nan[32:].any()
    assert not torch.isnan(vd).any()


@pytest.mark.parametrize("ks,vs", [(0.25, 4.0), (2.0 ** 20, 2.0 ** -20)])
def test_cache_scales(dev, ks, vs):
    g = torch.Generator().manual_seed(5)
    k = (torch.randn(9, 2, 128, generator=g) * ks).to(BF16)
    v = (torch.randn(9, 2, 128, generator=g) * vs).to(BF16)
    pool = _capi.fp4_pool(1, 2, 16, 128, dev)
    rows = torch.arange(9)
    _capi.kv_append_fp4(k=k.to(dev), v=v.to(dev), pool=pool, slot_rows=rows.to(dev), page_size=16,
                        k_scale=ks, v_scale=vs)
    kd, vd = _capi.gather_kv_rows_fp4(pool, rows.to(dev), page_size=16, dtype=BF16, k_scale=ks,
                                      v_scale=vs)
    assert np.array_equal(_np(kd), fp4.values(*fp4.quantise(_np(k) / ks)) * ks)
    assert np.array_equal(_np(vd), fp4.values(*fp4.quantise(_np(v) / vs)) * vs)


def _near_border(x, err):
    """Elements of x [.., D] whose code may differ when x is off by err (same shape)."""
    b, e = x.reshape(*x.shape[:-1], -1, 16), err.reshape(*x.shape[:-1], -1, 16)
    amax, emax = np.abs(b).max(-1) / 6, e.max(-1) / 6
    mid = (fp4.E4M3[1:] + fp4.E4M3[:-1]) / 2
    scale = (np.abs(amax[..., None] - mid) <= emax[..., None]).any(-1)
    s = fp4.e4m3_values(fp4.quantise(x)[1])[..., None]
    mid = (fp4.E2M1[1:] + fp4.E2M1[:-1]) / 2
    code = (np.abs(np.abs(b)[..., None] - s[..., None] * mid) <= e[..., None]).any(-1)
    return (code | scale[..., None]).reshape(x.shape)


@pytest.mark.parametrize("d,hq,hkv,dtype,norm,rope", [
    (128, 4, 2, BF16, True, True), (128, 3, 3, FP16, False, True), (64, 5, 1, BF16, True, False),
    (256, 2, 2, FP16, True, True), (64, 2, 2, FP16, False, True), (256, 4, 2, BF16, False, True)])
def test_norm_and_rotation(dev, d, hq, hkv, dtype, norm, rope):
    g = torch.Generator().manual_seed(d + hq)
    n, page = 21, 16
    # q, k and v are column blocks of one wider projection output
    qkv = torch.randn(n, (hq + 2 * hkv) * d + 8, generator=g).to(dtype).to(dev)
    q, k, v = (t.view(n, -1, d) for t in qkv[:, :(hq + 2 * hkv) * d].split(
        [hq * d, hkv * d, hkv * d], 1))
    qw = kw = cos = sin = None
    if norm:
        qw, kw = ((1 + 0.3 * torch.randn(2, d, generator=g)).to(dtype).to(dev))
    if rope:
        ang = torch.rand(n, d // 2, generator=g) * 6.3
        cos = torch.cat([ang.cos()] * 2, -1).to(dtype).to(dev)
        sin = torch.cat([ang.sin()] * 2, -1).to(dtype).to(dev)
    pool = _capi.fp4_pool(3, hkv, page, d, dev)
    rows = torch.randperm(3 * page, generator=g)[:n].to(dev)
    q_out = torch.full((n, hq + 1, d), 7.0, dtype=dtype, device=dev)[:, :hq]  # a wider buffer's view
    _capi.kv_append_fp4(q=q, k=k, v=v, q_out=q_out, q_norm_w=qw, k_norm_w=kw, eps=1e-6, cos=cos,
                        sin=sin, pool=pool, slot_rows=rows, page_size=page)
    kd, vd = _capi.gather_kv_rows_fp4(pool, rows, page_size=page, dtype=dtype)
    assert (q_out._base[:, hq:] == 7).all()

    def turned(x, w):
        """The row and a bound on what fp32 may add to it."""
        x, size = _np(x), np.abs(_np(x))
        if w is not None:
            f = _np(w) / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)
            x, size = x * f, size * np.abs(f)
        if cos is not None:
            c, s = _np(cos)[:, None], _np(sin)[:, None]
            h = d // 2
            rot = np.concatenate([-x[..., h:], x[..., :h]], -1)
            size = size * np.abs(c) + np.concatenate([size[..., h:], size[..., :h]], -1) * np.abs(s)
            x = x * c + rot * s
        return x, size * 2e-5

    qe, q_err = turned(q, qw)
    half = torch.finfo(dtype).eps / 2
    assert (np.abs(_np(q_out) - qe) <= np.abs(qe) * half * 1.001 + 2 * q_err + 2.0 ** -25).all()
    ke, k_err = turned(k, kw)
    near = _near_border(ke, k_err)
    assert near.mean() < 0.02
    want = fp4.values(*fp4.quantise(ke))
    assert np.array_equal(_np(kd)[~near], want[~near])
    assert np.array_equal(_np(vd), fp4.values(*fp4.quantise(_np(v))))


def test_append_without_q_and_bad_rows(dev):
    d, page = 128, 16
    x = torch.ones(3, 2, d, dtype=BF16, device=dev)
    pool = _capi.fp4_pool(2, 2, page, d, dev)
    rows = torch.tensor([5, 2 * page, 1 << 40], device=dev)  # the last two are outside the pool
    _capi.kv_append_fp4(k=x, v=x, pool=pool, slot_rows=rows, page_size=page)
    assert _capi.device_status(dev) == _capi.DEV_BAD_PAGE
    kd, _ = _capi.gather_kv_rows_fp4(pool, rows, page_size=page, dtype=BF16)
    assert _capi.device_status(dev) == _capi.DEV_BAD_PAGE
    # 1 reads back as 6 e4m3(1/6) = 6 * 0.171875
    assert np.array_equal(_np(kd[0]), fp4.values(*fp4.quantise(_np(x[0])))) and not kd[1:].any()
    written = (pool != 0).flatten(1).any(1).tolist()
    assert written == [True, False]


# ------------------------------------------------------------------ attention --
def _problem(dev, lens, hq, hkv, d, page, dtype, seed, k_scale=1.0, v_scale=1.0):
    """A pool filled with NaN scales outside the sequences' rows, K/V appended by the kernel."""
    g = torch.Generator().manual_seed(seed)
    b = len(lens)
    maxp = max(1, max(-(-n // page) for n in lens))
    pages = sum(-(-n // page) for n in lens) + 3
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((b, maxp), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(lens):
        m = -(-n // page)
        table[i, :m] = order[at:at + m]
        at += m
    pool = torch.full((pages, hkv, page // 16, 18 * d), 0x7F, dtype=torch.uint8, device=dev)
    total = sum(lens)
    k = (torch.randn(max(total, 1), hkv, d, generator=g) * k_scale).to(dtype)
    v = (torch.randn(max(total, 1), hkv, d, generator=g) * v_scale + 0.3).to(dtype)
    rows = [int(table[i, t // page]) * page + t % page for i, n in enumerate(lens) for t in range(n)]
    if rows:
        r = torch.tensor(rows, device=dev)
        for s in range(0, total, 4096):
            e = min(total, s + 4096)
            _capi.kv_append_fp4(k=k[s:e].to(dev), v=v[s:e].to(dev), pool=pool, slot_rows=r[s:e],
                                page_size=page, k_scale=k_scale, v_scale=v_scale)
    kd = fp4.values(*fp4.quantise(_np(k) / k_scale)) * k_scale
    vd = fp4.values(*fp4.quantise(_np(v) / v_scale)) * v_scale
    q = torch.randn(b, hq, d, generator=g).to(dtype)
    cut = np.cumsum([0] + list(lens))
    kv = [(kd[cut[i]:cut[i + 1]], vd[cut[i]:cut[i + 1]]) for i in range(b)]
    return q.to(dev), pool, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), kv


def _check_attention(q, kv, out, lse, scale, softcap=0.0, mask=None, rows=None):
    qn, o, l = _np(q), _np(out), lse.double().cpu().numpy()
    half_out = torch.finfo(out.dtype).eps / 2
    d = qn.shape[-1]
    for b in (range(len(kv)) if rows is None else rows):
        k, v = kv[b]
        m = None if mask is None else mask[b][:k.shape[0]]
        want, wl, size = fp4.attention(qn[b], k, v, scale, softcap, m)
        if not np.isfinite(wl).all():
            assert (o[b] == 0).all() and (l[b] == -np.inf).all()
            continue
        group = qn.shape[1] // k.shape[1]
        kk = np.repeat(k, group, axis=1)
        terms = np.abs(kk * qn[b][None]).sum(-1).max(0) * abs(scale)  # sum |q k|, largest key
        # one fp32 rounding per term of the product, score rounding and exp2 after it
        delta = terms * d * 2.0 ** -23 + (np.abs(wl) + terms + 20) * 2.0 ** -22
        if m is not None:
            fin = m[np.isfinite(m)]
            delta = delta + (np.abs(fin[np.abs(fin) < 1e30]).max(initial=0.0)) * 2.0 ** -23
        p_half = 2.0 ** -11          # P in fp16
        # P below fp16's normal range keeps absolute steps (the running maximum may lag by 2^8)
        tiny = k.shape[0] * 2.0 ** -25 * np.abs(v).max()
        tol = (size * (p_half + 2 * delta[:, None]) + np.abs(want) * half_out * 1.001 + tiny
               + 2.0 ** -25)
        bad = np.abs(o[b] - want) > tol
        assert not bad.any(), (b, np.abs(o[b] - want).max(), tol.min())
        assert (np.abs(l[b] - wl) <= delta + 1e-6 * (1 + np.abs(wl))).all(), (b, l[b] - wl)


CASES = [
    # lens, hq, hkv, d, page, dtype, softcap, k_scale, v_scale
    ([1], 8, 8, 128, 16, BF16, 0.0, 1.0, 1.0),
    ([0, 1, 15, 16, 17, 33], 8, 2, 128, 16, BF16, 0.0, 1.0, 1.0),
    ([0], 4, 4, 64, 16, FP16, 0.0, 1.0, 1.0),
    ([700, 64, 3], 40, 8, 128, 64, BF16, 0.0, 1.0, 1.0),
    ([129, 1000], 12, 12, 128, 48, FP16, 0.0, 0.25, 4.0),
    ([257, 30], 32, 2, 128, 16, BF16, 0.0, 1.0, 1.0),        # sixteen heads share a KV head
    ([511, 5], 27, 3, 64, 32, FP16, 0.0, 1.0, 0.5),          # nine
    ([300, 77], 16, 8, 256, 32, BF16, 50.0, 0.5, 2.0),
    ([200, 18], 32, 2, 256, 16, FP16, 0.0, 1.0, 1.0),
    ([4099], 5, 1, 128, 16, BF16, 0.0, 1.0, 1.0),            # one pair over many CTAs
    ([2500, 900, 31], 7, 1, 64, 16, BF16, 20.0, 1.0, 1.0),
    ([4099, 5], 4, 1, 128, 16, FP16, 0.0, 1.0, 1.0),         # fp16, up to four heads a KV head
    ([1500, 203, 0], 6, 2, 64, 16, FP16, 30.0, 1.0, 1.0),
    ([310, 77], 4, 2, 256, 32, FP16, 0.0, 0.5, 2.0),
    ([900, 33], 10, 2, 128, 16, FP16, 0.0, 1.0, 1.0),        # five
]


@pytest.mark.parametrize("case", CASES, ids=range(len(CASES)))
def test_decode_attention(dev, case):
    lens, hq, hkv, d, page, dtype, cap, ks, vs = case
    q, pool, table, kl, kv = _problem(dev, lens, hq, hkv, d, page, dtype, 3, ks, vs)
    lse = torch.empty(len(lens), hq, device=dev)
    kw = dict(num_kv_heads=hkv, page_size=page, scale=d ** -0.5, softcap=cap, k_scale=ks, v_scale=vs)
    out, _ = _capi.paged_decode_attention_fp4(q, pool, table, kl, lse=lse, **kw)
    assert _capi.device_status(dev) == 0
    _check_attention(q, kv, out, lse, d ** -0.5, cap)
    # a grid cut to the length: the same sums in another split, within the same bounds
    lse2 = torch.empty_like(lse)
    out2, _ = _capi.paged_decode_attention_fp4(q, pool, table, kl, lse=lse2,
                                               max_kv_len_hint=max(max(lens), 1), **kw)
    _check_attention(q, kv, out2, lse2, d ** -0.5, cap)


@pytest.mark.parametrize("mask_dtype", [torch.float32, BF16, FP16])
@pytest.mark.parametrize("low", ["inf", "lowest"])
def test_masks(dev, mask_dtype, low):
    lens, hq, hkv, d, page = [100, 333, 40, 1], 8, 4, 128, 16
    q, pool, table, kl, kv = _problem(dev, lens, hq, hkv, d, page, BF16, 11)
    g = torch.Generator().manual_seed(2)
    mask = torch.randn(4, 340, generator=g).to(mask_dtype)
    bottom = float("-inf") if low == "inf" else torch.finfo(mask_dtype).min
    mask[0, :70] = bottom            # left padding, a whole tile among it
    mask[1, torch.randperm(333, generator=g)[:200]] = bottom
    mask[2, :] = bottom              # leaves the row nothing (or all keys alike)
    lse = torch.empty(4, hq, device=dev)
    out, _ = _capi.paged_decode_attention_fp4(q, pool, table, kl, num_kv_heads=hkv, page_size=page,
                                              scale=0.1, mask=mask.to(dev), lse=lse)
    m = _np(mask)
    if low == "lowest" and mask_dtype != FP16:
        # adding the scores to a mask of -3.4e38 leaves the mask: a plain mean of V
        row = _np(out)[2]
        mean = np.repeat(kv[2][1].mean(0), 2, axis=0)
        size = np.repeat(np.abs(kv[2][1]).mean(0), 2, axis=0)
        assert (np.abs(row - mean) <= size * 2.0 ** -10 + np.abs(mean) * 2.0 ** -8).all()
        assert np.allclose(lse[2].double().cpu().numpy(), bottom, rtol=1e-6)
        _check_attention(q, kv, out, lse, 0.1, 0.0, m, rows=[0, 1, 3])
    else:
        _check_attention(q, kv, out, lse, 0.1, 0.0, m)


def test_nan_pages_under_an_inf_mask(dev):
    lens, hq, hkv, d, page = [90], 4, 1, 128, 16
    q, pool, table, kl, kv = _problem(dev, lens, hq, hkv, d, page, BF16, 13)
    pool[table[0, 1].item()] = 0x7F   # tokens 16..31: NaN scales
    mask = torch.zeros(1, 90)
    mask[0, 16:32] = float("-inf")
    mask[0, 60] = float("-inf")
    lse = torch.empty(1, hq, device=dev)
    out, _ = _capi.paged_decode_attention_fp4(q, pool, table, kl, num_kv_heads=hkv, page_size=page,
                                              scale=0.1, mask=mask.to(dev), lse=lse)
    _check_attention(q, kv, out, lse, 0.1, 0.0, _np(mask))


def test_a_mask_shorter_than_the_keys_cuts_them(dev):
    lens, hq, hkv, d, page = [90, 20], 8, 2, 128, 16
    q, pool, table, kl, kv = _problem(dev, lens, hq, hkv, d, page, BF16, 19)
    mask = torch.randn(2, 50, generator=torch.Generator().manual_seed(4))
    lse = torch.empty(2, hq, device=dev)
    # (the mask lies across its memory, so that the call has to lay it out anew)
    across = mask.t().contiguous().to(dev).t()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    out, _ = _capi.paged_decode_attention_fp4(q, pool, table, kl, num_kv_heads=hkv, page_size=page,
                                              scale=0.1, mask=across, lse=lse, stream=side)
    side.synchronize()
    assert _capi.device_status(dev) == _capi.DEV_BAD_PAGE
    kv[0] = tuple(x[:50] for x in kv[0])
    _check_attention(q, kv, out, lse, 0.1, 0.0, _np(mask))


def test_no_tokens(dev):
    pool = _capi.fp4_pool(2, 2, 16, 64, dev)
    none = torch.empty(0, 2, 64, dtype=BF16, device=dev)
    rows = torch.empty(0, dtype=torch.long, device=dev)
    _capi.kv_append_fp4(k=none, v=none, q=none, q_out=none, pool=pool, slot_rows=rows, page_size=16)
    k, v = _capi.gather_kv_rows_fp4(pool, rows, page_size=16, dtype=FP16)
    assert k.shape == v.shape == (0, 2, 64) and not pool.any()


def test_large_and_tiny_queries(dev):
    """bf16 queries outside fp16's range, and scores whose maximum climbs along the sequence."""
    lens, hq, hkv, d, page = [400], 4, 2, 128, 16
    q, pool, table, kl, kv = _problem(dev, lens, hq, hkv, d, page, BF16, 17)
    q[0, 0] *= 2.0 ** 20
    q[0, 1] *= 2.0 ** -30
    q[0, 2] = 0
    scale = 2.0 ** -20
    lse = torch.empty(1, hq, device=dev)
    out, _ = _capi.paged_decode_attention_fp4(q, pool, table, kl, num_kv_heads=hkv, page_size=page,
                                              scale=scale, lse=lse)
    _check_attention(q, kv, out, lse, scale)
    # keys in rising order of their score with head 3: the maximum moves at every tile
    n, g = 400, 2
    s = kv[0][0][:, 1] @ _np(q)[0, 3]
    order = np.argsort(s)
    rows = [int(table[0, t // page]) * page + t % page for t in range(n)]
    k = torch.from_numpy(kv[0][0][order]).to(BF16).to(dev)
    v = torch.from_numpy(kv[0][1][order]).to(BF16).to(dev)
    _capi.kv_append_fp4(k=k, v=v, pool=pool, slot_rows=torch.tensor(rows, device=dev),
                        page_size=page)
    kv2 = [tuple(fp4.values(*fp4.quantise(_np(x))) for x in (k, v))]
    out, _ = _capi.paged_decode_attention_fp4(q, pool, table, kl, num_kv_heads=hkv, page_size=page,
                                              scale=1.0, lse=lse)
    _check_attention(q[:, 3:], [(kv2[0][0][:, 1:], kv2[0][1][:, 1:])], out[:, 3:], lse[:, 3:], 1.0)


def test_negative_scale(dev):
    q, pool, table, kl, kv = _problem(dev, [130], 4, 2, 64, 16, BF16, 19)
    lse = torch.empty(1, 4, device=dev)
    out, _ = _capi.paged_decode_attention_fp4(q, pool, table, kl, num_kv_heads=2, page_size=16,
                                              scale=-0.2, lse=lse)
    _check_attention(q, kv, out, lse, -0.2)


def test_strided_tensors_other_stream_and_other_place(dev):
    lens, hq, hkv, d, page = [333, 90], 8, 2, 128, 16
    q, pool, table, kl, kv = _problem(dev, lens, hq, hkv, d, page, FP16, 23)
    kw = dict(num_kv_heads=hkv, page_size=page, scale=0.09)
    ref, _ = _capi.paged_decode_attention_fp4(q, pool, table, kl, **kw)
    # q and out as views of wider buffers, a table with longer rows
    wide = torch.zeros(2, hq + 3, d + 16, dtype=FP16, device=dev)
    wide[:, 1:hq + 1, 8:d + 8] = q
    buf = torch.full((2, hq, 2 * d), 5.0, dtype=FP16, device=dev)
    long_table = torch.full((2, table.shape[1] + 7), 1 << 30, dtype=torch.int32, device=dev)
    long_table[:, :table.shape[1]] = table
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    out, _ = _capi.paged_decode_attention_fp4(wide[:, 1:hq + 1, 8:d + 8], pool, long_table, kl,
                                              out=buf[:, :, :d], stream=s, **kw)
    s.synchronize()
    assert torch.equal(buf[:, :, :d], ref) and (buf[:, :, d:] == 5).all()
    # every page at another place of the pool: the same bits
    perm = torch.randperm(pool.shape[0], device=dev)
    moved = torch.empty_like(pool)
    moved[perm] = pool
    t2 = torch.where(table >= 0, perm[table.clamp(min=0).long()].int(), table)
    again, _ = _capi.paged_decode_attention_fp4(q, moved, t2, kl, **kw)
    assert torch.equal(again, ref)
    assert _capi.device_status(dev) == 0


def test_bad_page_entries_and_lengths_are_reported(dev):
    q, pool, table, kl, _ = _problem(dev, [100], 4, 2, 128, 16, BF16, 29)
    kw = dict(num_kv_heads=2, page_size=16, scale=0.09)
    bad = table.clone()
    bad[0, 2] = pool.shape[0]
    _capi.paged_decode_attention_fp4(q, pool, bad, kl, **kw)
    assert _capi.device_status(dev) == _capi.DEV_BAD_PAGE
    _capi.paged_decode_attention_fp4(q, pool, table, kl + 100, **kw)  # longer than the table
    assert _capi.device_status(dev) == _capi.DEV_BAD_PAGE
    _capi.paged_decode_attention_fp4(q, pool, table, kl - 200, **kw)  # negative: empty
    assert _capi.device_status(dev) == 0


def test_two_captured_graphs_and_eager_calls_interleave(dev):
    probs = [_problem(dev, lens, 8, 2, 128, 16, BF16, s) for lens, s in (([700, 20], 31), ([90, 1500], 37))]
    kw = dict(num_kv_heads=2, page_size=16, scale=0.09)
    refs = [_capi.paged_decode_attention_fp4(*p[:4], **kw)[0].clone() for p in probs]
    outs = [torch.empty_like(p[0]) for p in probs]
    graphs = []
    for p, o in zip(probs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            _capi.paged_decode_attention_fp4(*p[:4], out=o, **kw)
        graphs.append(g)
    torch.cuda.synchronize(dev)
    streams = [torch.cuda.Stream(dev) for _ in probs]
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize(dev)
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = _capi.paged_decode_attention_fp4(*probs[0][:4], **kw)[0]
        torch.cuda.synchronize(dev)
        assert torch.equal(eager, refs[0])
        for o, r in zip(outs, refs):
            assert torch.equal(o, r)


def test_decode_overlap_after_the_append(dev):
    """A captured step: append, then attention as its programmatic dependent."""
    lens, hq, hkv, d, page = [47, 16, 200], 8, 4, 128, 16
    q, pool, table, kl, _ = _problem(dev, lens, hq, hkv, d, page, BF16, 41)
    g = torch.Generator().manual_seed(43)
    k = torch.randn(3, hkv, d, generator=g).to(BF16).to(dev)
    # the next row of each sequence (the second starts a page of its own)
    rows = torch.tensor([int(table[0, 2]) * 16 + 15, int(table[1, 0]) * 16 + 15,
                         int(table[2, 12]) * 16 + 7], device=dev)
    kl1 = torch.tensor([48, 16, 200], dtype=torch.int32, device=dev)
    kw = dict(num_kv_heads=hkv, page_size=page, scale=0.09)
    fresh = pool.clone()
    _capi.kv_append_fp4(k=k, v=k, pool=fresh, slot_rows=rows, page_size=page)
    ref, _ = _capi.paged_decode_attention_fp4(q, fresh, table, kl1, **kw)
    out = torch.empty_like(ref)
    graph = torch.cuda.CUDAGraph()
    with _capi.decode_overlap(), torch.cuda.graph(graph):
        _capi.kv_append_fp4(k=k, v=k, pool=pool, slot_rows=rows, page_size=page)
        _capi.paged_decode_attention_fp4(q, pool, table, kl1, out=out, **kw)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize(dev)
        assert torch.equal(out, ref)


def test_pages_beyond_four_gigabytes(dev):
    """Byte offsets above 2^32 and pool rows above 2^31 / page elements."""
    hkv, d, page, lens = 8, 128, 64, [300]
    per = _capi.fp4_page_bytes(hkv, page, d)
    pages = (1 << 32) // per + 40
    pool = torch.empty(pages, hkv, page // 16, 18 * d, dtype=torch.uint8, device=dev)
    g = torch.Generator().manual_seed(47)
    table = torch.tensor([[pages - 1, pages - 7, 0, pages - 3, 12]], dtype=torch.int32)
    k = torch.randn(300, hkv, d, generator=g).to(BF16)
    v = torch.randn(300, hkv, d, generator=g).to(BF16)
    rows = torch.tensor([int(table[0, t // page]) * page + t % page for t in range(300)], device=dev)
    _capi.kv_append_fp4(k=k.to(dev), v=v.to(dev), pool=pool, slot_rows=rows, page_size=page)
    kd, vd = _capi.gather_kv_rows_fp4(pool, rows, page_size=page, dtype=BF16)
    kv = [tuple(fp4.values(*fp4.quantise(_np(x))) for x in (k, v))]
    assert np.array_equal(_np(kd), kv[0][0]) and np.array_equal(_np(vd), kv[0][1])
    q = torch.randn(1, 16, d, generator=g).to(BF16).to(dev)
    lse = torch.empty(1, 16, device=dev)
    out, _ = _capi.paged_decode_attention_fp4(q, pool, table.to(dev),
                                              torch.tensor([300], dtype=torch.int32, device=dev),
                                              num_kv_heads=hkv, page_size=page, scale=0.09, lse=lse)
    _check_attention(q, kv, out, lse, 0.09)
    del pool
    torch.cuda.empty_cache()


def test_many_sequences(dev):
    """More sequences than CTAs, most of them short, some empty."""
    lens = [(i * 7) % 40 for i in range(300)]
    q, pool, table, kl, kv = _problem(dev, lens, 4, 2, 64, 16, FP16, 53)
    lse = torch.empty(300, 4, device=dev)
    out, _ = _capi.paged_decode_attention_fp4(q, pool, table, kl, num_kv_heads=2, page_size=16,
                                              scale=0.125, lse=lse)
    _check_attention(q, kv, out, lse, 0.125)
    assert _capi.device_status(dev) == 0


def test_wrapper_refusals(dev):
    q, pool, table, kl, _ = _problem(dev, [20], 4, 2, 128, 16, BF16, 59)
    kw = dict(num_kv_heads=2, page_size=16, scale=0.09)
    call = _capi.paged_decode_attention_fp4
    for bad in (lambda: call(q, pool.float(), table, kl, **kw),
                lambda: call(q, pool[:, :1], table, kl, **kw),
                lambda: call(q, pool, table.long(), kl, **kw),
                lambda: call(q, pool, table, kl.cpu(), **kw),
                lambda: call(q, pool, table.t(), kl, **kw),
                lambda: call(q.float(), pool, table, kl, **kw),
                lambda: call(q, pool, table, kl, out=q[:, :2], **kw),
                lambda: call(q, pool, table, kl, mask=torch.zeros(3, 20, device=dev), **kw),
                lambda: call(q, pool, table, kl, lse=torch.empty(1, 3, device=dev), **kw),
                lambda: call(q, pool, table, kl, num_kv_heads=2, page_size=32, scale=0.09)):
        with pytest.raises(_capi.HelmError):
            bad()
    x = torch.zeros(2, 2, 128, dtype=BF16, device=dev)
    rows = torch.tensor([0, 1], device=dev)
    for kwargs in (dict(k=x, v=x[:1]), dict(k=x, v=x.half()), dict(k=x, v=x, q=x),
                   dict(k=x, v=x, cos=x[:, 0]), dict(k=x, v=x, k_norm_w=x[0, 0, :64]),
                   dict(k=x, v=x, slot_rows=rows.int()), dict(k=x, v=x, k_scale=3.0)):
        with pytest.raises(_capi.HelmError):
            _capi.kv_append_fp4(**{**dict(pool=pool, slot_rows=rows, page_size=16), **kwargs})
