"""The 4-bit format's oracle against its definition, and the refusals of the
4-bit entry points, the step tables and the sampler (no GPU needed: refused
calls return before any device work)."""
import ctypes

import numpy as np
import pytest
import torch

from helm_b200 import _capi
from oracle import fp4, serving

OK, INVALID, UNSUPPORTED, WORKSPACE, ALIGN = 0, 1, 2, 4, 5
BF16, FP16, FP32 = _capi.DTYPE_BF16, _capi.DTYPE_FP16, _capi.DTYPE_FP32
P16 = 0x10000  # aligned placeholder address (never dereferenced)
P256 = 0x100000
F = ctypes.c_float


@pytest.mark.parametrize("d", [64, 128, 256])
def test_tile_layout_covers_every_byte_once(d):
    seen = np.concatenate([np.concatenate(fp4.tile_bytes(d, t)) for t in range(16)])
    assert np.array_equal(np.sort(seen), np.arange(18 * d))


def test_scale_table_is_torch_e4m3():
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double().numpy()
    got = fp4.e4m3_values(codes.numpy())
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)])


def test_quantise_picks_the_nearest_level():
    g = np.random.default_rng(0)
    x = g.standard_normal((50, 64)) * np.exp(g.uniform(-6, 6, (50, 1)))
    codes, s8 = fp4.quantise(x)
    s = fp4.e4m3_values(s8)
    # brute force over all scales and levels
    amax = np.abs(x.reshape(50, 4, 16)).max(-1) / 6
    assert np.allclose(np.abs(s - np.minimum(amax, 448)),
                       np.abs(fp4.E4M3 - np.minimum(amax, 448)[..., None]).min(-1))
    v = fp4.values(codes, s8).reshape(50, 4, 16)
    levels = np.concatenate([fp4.E2M1, -fp4.E2M1]) * s[..., None, None]
    best = np.abs(x.reshape(50, 4, 16, 1) - levels).min(-1)
    assert np.allclose(np.abs(x.reshape(50, 4, 16) - v), best, rtol=0, atol=1e-12)


def test_quantise_ties_zeros_and_non_finite():
    x = np.zeros((1, 16))
    x[0, :9] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25]
    codes, s8 = fp4.quantise(x)
    assert s8[0, 0] == 0x38  # 1.0
    assert codes[0, :9].tolist() == [7, 0, 2, 2, 4, 4, 6, 6, 8]  # ties to even codes
    assert fp4.quantise(np.zeros((1, 16)))[1][0, 0] == 0
    x[0, 3] = np.inf
    codes, s8 = fp4.quantise(x)
    assert s8[0, 0] == 0x7E and codes[0, 3] == 7
    x[0, 3] = np.nan
    assert fp4.quantise(x)[1][0, 0] == 0x7F


def test_rows_round_trip_through_the_tiles():
    g = np.random.default_rng(1)
    for d in (64, 128, 256):
        pool = np.full((3, 2, 3, 18 * d), 0xAB, np.uint8)
        rows = [0, 47, 17, -1, 96 + 5, 48 + 30]
        k, v = g.standard_normal((2, len(rows), 2, d))
        fp4.write_rows(pool, rows, k, v, 48)
        kd, vd = fp4.read_rows(pool, rows, 48)
        for x, y in ((k, kd), (v, vd)):
            want = fp4.values(*fp4.quantise(x))
            want[3] = 0
            assert np.array_equal(y, want)


def test_page_bytes():
    assert _capi.fp4_page_bytes(8, 16, 128) == 8 * 2304
    assert _capi.fp4_page_bytes(2, 64, 64) == 2 * 4 * 1152
    for bad in ((8, 24, 128), (8, 16, 96), (0, 16, 128)):
        with pytest.raises(_capi.HelmError):
            _capi.fp4_page_bytes(*bad)


# ------------------------------------------------------------------ refusals --
def _append(**kw):
    a = dict(q=P16, q_st=6144, q_sh=128, k=P16, k_st=6144, k_sh=128, v=P16, v_st=6144, v_sh=128,
             qw=P16, kw=P16, cos=P16, sin=P16, rope_st=128, q_out=P16, qo_st=4096, qo_sh=128,
             pool=P16, pages=64, rows=P16, n=0, hq=32, hkv=8, d=128, page=16, dtype=BF16, ks=1.0,
             vs=1.0)
    a.update(kw)
    return _capi.lib().helm_kv_append_fp4(
        a["q"], a["q_st"], a["q_sh"], a["k"], a["k_st"], a["k_sh"], a["v"], a["v_st"], a["v_sh"],
        a["qw"], a["kw"], F(1e-6), a["cos"], a["sin"], a["rope_st"], a["q_out"], a["qo_st"],
        a["qo_sh"], a["pool"], a["pages"], a["rows"], a["n"], a["hq"], a["hkv"], a["d"], a["page"],
        a["dtype"], a["ks"], a["vs"], None)


def test_append_refusals():
    assert _append() == OK  # no tokens: nothing to do
    assert _append(k=None) == INVALID
    assert _append(pool=None) == INVALID
    assert _append(rows=None) == INVALID
    assert _append(q_out=None) == INVALID
    assert _append(sin=None) == INVALID
    assert _append(n=-1) == INVALID
    assert _append(pages=0) == INVALID
    assert _append(ks=0.75) == INVALID            # not a power of two
    assert _append(vs=0.0) == INVALID
    assert _append(vs=-1.0) == INVALID
    assert _append(vs=float("inf")) == INVALID
    assert _append(ks=float("nan")) == INVALID
    assert _append(d=96) == UNSUPPORTED
    assert _append(page=24) == UNSUPPORTED
    assert _append(dtype=FP32) == UNSUPPORTED
    assert _append(q=P16 + 8) == ALIGN
    assert _append(k_st=6148) == ALIGN
    assert _append(pool=P16 + 4) == ALIGN


def _gather(**kw):
    a = dict(pool=P16, pages=64, rows=P16, k=P16, st=1024, sh=128, v=P16, n=0, hkv=8, d=128,
             page=16, dtype=BF16, ks=1.0)
    a.update(kw)
    return _capi.lib().helm_gather_kv_rows_fp4(
        a["pool"], a["pages"], a["rows"], a["k"], a["st"], a["sh"], a["v"], a["st"], a["sh"],
        a["n"], a["hkv"], a["d"], a["page"], a["dtype"], a["ks"], 1.0, None)


def test_gather_refusals():
    assert _gather() == OK
    assert _gather(k=None) == INVALID
    assert _gather(rows=None) == INVALID
    assert _gather(ks=3.0) == INVALID
    assert _gather(hkv=0) == INVALID
    assert _gather(d=80) == UNSUPPORTED
    assert _gather(dtype=FP32) == UNSUPPORTED
    assert _gather(sh=132) == ALIGN
    assert _gather(v=P16 + 2) == ALIGN


def _decode(**kw):
    a = dict(q=P16, q_sb=4096, q_sh=128, pool=P16, pages=64, pt=P16, pt_sb=19, maxp=19, lens=P16,
             mask=None, mask_dtype=0, mask_len=304, out=P16, ws=P256, ws_bytes=1 << 30, batch=2,
             hq=32, hkv=8, d=128, page=16, dtype=BF16, ks=1.0, vs=1.0)
    a.update(kw)
    return _capi.lib().helm_paged_decode_attention_fp4(
        a["q"], a["q_sb"], a["q_sh"], a["pool"], a["pages"], a["pt"], a["pt_sb"], a["maxp"],
        a["lens"], a["mask"], a["mask_dtype"], 0, a["mask_len"], a["out"], 4096, 128, None, a["ws"],
        a["ws_bytes"], a["batch"], a["hq"], a["hkv"], a["d"], a["page"], a["dtype"], 0.088, 0.0,
        a["ks"], a["vs"], 0, None)


def test_decode_refusals():
    assert _decode(q=None) == INVALID
    assert _decode(ws=None) == INVALID
    assert _decode(batch=0) == INVALID
    assert _decode(hq=30) == INVALID
    assert _decode(ks=1.5) == INVALID
    assert _decode(mask=P16, mask_dtype=7) == INVALID
    assert _decode(mask=P16, mask_dtype=BF16, mask_len=-1) == INVALID
    assert _decode(hq=136) == UNSUPPORTED       # GQA group of 17
    assert _decode(batch=2049) == UNSUPPORTED
    assert _decode(d=96) == UNSUPPORTED
    assert _decode(page=8) == UNSUPPORTED
    assert _decode(dtype=FP32) == UNSUPPORTED
    assert _decode(maxp=1 << 27) == UNSUPPORTED  # token positions must fit 31 bits
    assert _decode(q=P16 + 2) == ALIGN
    assert _decode(q_sh=129) == ALIGN
    assert _decode(pool=P16 + 8) == ALIGN
    assert _decode(ws=P256 + 16) == ALIGN
    assert _decode(ws_bytes=16) == WORKSPACE


def _tables(**kw):
    a = dict(past=P16, new=P16, table=P16, sb=10, maxp=10, free=P16, cap=100, count=P16, cout=P16,
             kv=P16, cu=P16, rows=P16, batch=4, page=16, n=8)
    a.update(kw)
    return _capi.lib().helm_build_step_tables(
        a["past"], a["new"], a["table"], a["sb"], a["maxp"], a["free"], a["cap"], a["count"],
        a["cout"], a["kv"], a["cu"], None, None, a["rows"], a["batch"], a["page"], a["n"], None)


def test_step_table_refusals():
    for name in ("past", "new", "table", "free", "count", "cout", "kv", "cu", "rows"):
        assert _tables(**{name: None}) == INVALID, name
    assert _tables(batch=0) == INVALID
    assert _tables(page=0) == INVALID
    assert _tables(maxp=0) == INVALID
    assert _tables(sb=9) == INVALID
    assert _tables(cap=-1) == INVALID
    assert _tables(n=-1) == INVALID
    assert _tables(batch=8193) == UNSUPPORTED
    assert _tables(batch=8192, maxp=1 << 18, sb=1 << 18) == UNSUPPORTED
    assert _tables(page=1 << 20, maxp=1 << 11, sb=1 << 11) == UNSUPPORTED


def _sample(**kw):
    a = dict(logits=P16, st=1000, dtype=BF16, u=P16, ids=P16, batch=2, vocab=1000)
    a.update(kw)
    return _capi.lib().helm_sample_tokens(a["logits"], a["st"], a["dtype"], a["u"], None, None,
                                          None, None, a["ids"], None, a["batch"], a["vocab"], None)


def test_sample_refusals():
    assert _sample(batch=0) == OK
    assert _sample(logits=None) == INVALID
    assert _sample(u=None) == INVALID
    assert _sample(ids=None) == INVALID
    assert _sample(vocab=0) == INVALID
    assert _sample(batch=-1) == INVALID
    assert _sample(vocab=(1 << 18) + 1) == UNSUPPORTED
    assert _sample(dtype=9) == UNSUPPORTED


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    rows = torch.zeros(2, dtype=torch.int64)
    pool = torch.zeros(1, 2, 1, 18 * 64, dtype=torch.uint8)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(_capi.HelmError, match="CUDA"):
        _capi.kv_append_fp4(k=x, v=x, pool=pool, slot_rows=rows, page_size=16)
    with pytest.raises(_capi.HelmError, match="CUDA"):
        _capi.gather_kv_rows_fp4(pool, rows, page_size=16, dtype=torch.bfloat16)
    with pytest.raises(_capi.HelmError, match="CUDA"):
        _capi.paged_decode_attention_fp4(x, pool, i.view(2, 1), i, num_kv_heads=2, page_size=16,
                                         scale=0.1)
    with pytest.raises(_capi.HelmError, match="CUDA"):
        _capi.build_step_tables(i, i, i.view(2, 1), i, i[:1], page_size=16, num_rows=2)
    with pytest.raises(_capi.HelmError, match="CUDA"):
        _capi.sample_tokens(torch.zeros(2, 8), torch.zeros(2))


# ------------------------------------------------- the oracles on small cases --
def test_step_tables_oracle_small_case():
    r = serving.step_tables([16, 0, 20, 5], [1, 3, -1, 0], [[4, 9], [9, 9], [7, 8], [2, 9]],
                            [1, 3, 9, 9], 2, 16, 6)
    # request 2 gives back 7 and 8; request 0 then takes 8, request 1 takes 7
    assert r["page_table"] == [[4, 8], [7, 9], [7, 8], [2, 9]]
    assert r["free_pages"] == [1, 3, 7, 8] and r["free_count"] == 2
    assert r["kv_lens"] == [17, 3, 0, 5] and r["cu_tokens"] == [0, 1, 4, 4, 4]
    assert r["slot_rows"] == [8 * 16, 7 * 16, 7 * 16 + 1, 7 * 16 + 2, -1, -1]
    assert not r["refused"]


def test_sampling_oracle_small_case():
    l = np.log([0.1, 0.4, 0.2, 0.3])
    assert [serving.sample(l, u)[0] for u in (0.05, 0.3, 0.6, 0.99)] == [0, 1, 2, 3]
    assert serving.sample(l, 0.99, top_k=2)[0] == 3
    assert serving.sample(l, 0.0, top_k=2)[0] == 1
    assert serving.sample(l, 0.99, top_p=0.65)[0] == 3  # 0.4 + 0.3
    assert serving.sample(l, 0.0, top_p=0.65)[0] == 1
    assert serving.sample(l, 0.5, min_p=0.9)[0] == 1
    assert serving.sample(l, 0.5, temperature=0)[0] == 1
    assert np.isclose(serving.sample(l, 0.05)[1], np.log(0.1))
