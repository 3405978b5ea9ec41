"""The token step of a server over a 4-bit KV cache, operator by operator: plain forms and cases.

Four operators, in the order a step uses them:

  tables  block table, slot rows and positions of a step's tokens from the requests' lengths
  append  per-head RMSNorm and rotary embedding of q and k, K and V quantised into the pages
          (and the rows read back as the values they stand for)
  attend  decode attention over the 4-bit pages
  sample  one token per row from the logits: temperature, top-k, top-p, min-p, given uniforms

The 4-bit format: 16 consecutive values of a head row share an e4m3 scale
s = e4m3(max|x| / 6), each value is the nearest e2m1 number (0, .5, 1, 1.5, 2, 3, 4, 6) to x / s.
A pool is uint8 [pages, KV heads, page_size / 16, 18 * D]; its last dimension is a tile of 16 tokens
(K codes, V codes, K scales, V scales), laid out as _tile_offsets() says.
"""
import math

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------ cases --
def listed():
    return [
        # a step of sixteen requests, one token each: nothing but latency
        dict(name="tables_decode16", kind="tables", batch=16, page=16, past=2048, chunk=0, spare=64),
        # a continuous-batching step: two thousand requests, every eighth with a prompt chunk, some leaving
        dict(name="tables_mixed2048", kind="tables", batch=2048, page=16, past=4096, chunk=509,
             spare=65536),
        # one token of each of sixteen sequences, as many KV heads as query heads (Llama-2-13B heads)
        dict(name="append_decode16_mha", kind="append", tokens=16, hq=40, hkv=40, d=128, page=16,
             dtype="fp16", norm=False, rope=True, k_scale=1.0, v_scale=1.0),
        # a prompt's rows (Qwen3-8B heads, QK-norm and rotary embedding)
        dict(name="append_prompt4096", kind="append", tokens=4096, hq=32, hkv=8, d=128, page=64,
             dtype="bf16", norm=True, rope=True, k_scale=1.0, v_scale=1.0),
        # a short context at batch 1 (Qwen3-0.6B heads): latency
        dict(name="attend_576", kind="attend", batch=1, hq=16, hkv=8, d=128, page=64, length=576,
             ragged=0, dtype="bf16", mask="none", softcap=0.0, k_scale=1.0, v_scale=1.0),
        # sixteen ragged sequences without head sharing (Llama-2-13B heads)
        dict(name="attend_b16_mha", kind="attend", batch=16, hq=40, hkv=40, d=128, page=16,
             length=2304, ragged=17, dtype="fp16", mask="none", softcap=0.0, k_scale=1.0,
             v_scale=1.0),
        # wide heads with soft-capping and left padding (a Gemma-2-shaped batch)
        dict(name="attend_d256_padded", kind="attend", batch=8, hq=16, hkv=8, d=256, page=32,
             length=4001, ragged=301, dtype="bf16", mask="low", softcap=50.0, k_scale=0.5,
             v_scale=2.0),
        # the decode call of four 32768-token sequences
        dict(name="attend_4x32k", kind="attend", batch=4, hq=32, hkv=8, d=128, page=16,
             length=32768, ragged=0, dtype="bf16", mask="none", softcap=0.0, k_scale=1.0,
             v_scale=1.0),
        # one 131072-token sequence (Qwen3-14B heads)
        dict(name="attend_128k", kind="attend", batch=1, hq=40, hkv=8, d=128, page=64,
             length=131072, ragged=0, dtype="bf16", mask="none", softcap=0.0, k_scale=1.0,
             v_scale=1.0),
        # one row of a large vocabulary, nucleus sampling
        dict(name="sample_1x152k", kind="sample", batch=1, vocab=151936, dtype="bf16", mode="top_p"),
        # a small batch over a small vocabulary, every filter at once, some rows greedy
        dict(name="sample_16x32k", kind="sample", batch=16, vocab=32000, dtype="fp32", mode="mixed"),
        # a full batch of a large vocabulary
        dict(name="sample_256x152k", kind="sample", batch=256, vocab=151936, dtype="bf16",
             mode="mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "append", "attend", "attend", "sample"])
    scales = dict(k_scale=rng.choice([0.25, 0.5, 1.0, 2.0]), v_scale=rng.choice([0.5, 1.0, 4.0]))
    if kind == "tables":
        batch = _log(rng, 1, 2048)
        chunk = rng.choice([0, _log(rng, 2, 509)])
        return dict(kind=kind, batch=batch, page=rng.choice([16, 32, 64]), past=_log(rng, 1, 4096),
                    chunk=chunk, spare=_log(rng, 1, 65536))
    if kind == "append":
        d = rng.choice([64, 128, 256])
        hkv = rng.choice([1, 2, 4, 5, 8])
        return dict(kind=kind, tokens=_log(rng, 1, 4096), hq=hkv * rng.choice([1, 2, 3, 4]), hkv=hkv,
                    d=64 if d == 256 and hkv > 4 else d, page=rng.choice([16, 48, 64]),
                    dtype=rng.choice(["bf16", "fp16"]), norm=rng.random() < 0.5,
                    rope=rng.random() < 0.7, **scales)
    if kind == "attend":
        d = rng.choice([64, 128, 128, 256])
        hkv = rng.choice([1, 2, 3, 4, 8])
        batch = _log(rng, 1, 64)
        most = max(2, min(131072, 4 * 32768 * 8 * 128 // (batch * hkv * d)))
        length = _log(rng, 1, most)
        return dict(kind=kind, batch=batch, hq=hkv * rng.randint(1, 16 if d < 256 else 8), hkv=hkv,
                    d=d, page=rng.choice([16, 48, 64]), length=length,
                    ragged=rng.choice([0, 1, max(1, length // (batch + 1))]),
                    dtype=rng.choice(["bf16", "fp16"]), mask=rng.choice(["none", "none", "low", "inf"]),
                    softcap=rng.choice([0.0, 0.0, 30.0]), **scales)
    return dict(kind=kind, batch=_log(rng, 1, 256), vocab=_log(rng, 900, 151936),
                dtype=rng.choice(["bf16", "fp16", "fp32"]),
                mode=rng.choice(["none", "top_k", "top_p", "min_p", "mixed"]))


# -------------------------------------------------------------- the 4-bit format --
def _tile_offsets(d, device):
    """Byte offsets in a tile of K codes [16, d/2], V codes [16, d/2], K scales and V scales
    [16, d/16].  Code byte i of a token holds dims 2i (low four bits) and 2i+1."""
    t = torch.arange(16, device=device)[:, None]
    row = t ^ (((t >> 1) & 2) | ((t >> 3) & 1))
    i = torch.arange(d // 2, device=device)[None]
    k16 = (i >> 4) ^ (4 * (t & 1) if d == 256 else 0 * t)
    kcode = row * (d // 2) + k16 * 16 + (i & 15)
    chunk = d // 16
    turn = {64: 0 * t, 128: 4 * ((t >> 2) & 1), 256: 2 * ((t >> 2) & 3)}[d]
    vcode = 8 * d + row * (d // 2) + ((i // chunk) ^ turn) * chunk + i % chunk
    g = torch.arange(d // 16, device=device)[None]
    c, k = {64: (g, 0 * g), 128: (g >> 1, g & 1), 256: ((g & 7) >> 1, (g & 1) | ((g >> 3) << 1))}[d]
    pair, second = ((t >> 2) << 1) | (t & 1), (t >> 1) & 1
    kscale = 16 * d + (pair * 4 + c) * (d // 32) + second * (d // 64) + k
    vscale = 17 * d + g * 16 + t
    return kcode, vcode, kscale, vscale


def _quantise(x):
    """x [..., d] fp32 -> (codes uint8 [..., d], scale bytes uint8 [..., d/16])."""
    b = x.unflatten(-1, (-1, 16))
    s = (b.abs().amax(-1) / 6.0).clamp(max=448.0).to(torch.float8_e4m3fn)
    r = b.double().abs() / s.double()[..., None]
    r = torch.where(s.float()[..., None] > 0, r, torch.zeros_like(r))
    # ties go to the even code
    c = ((r > 0.25).to(torch.uint8) + (r >= 0.75) + (r > 1.25) + (r >= 1.75) + (r > 2.5)
         + (r >= 3.5) + (r > 5.0))
    c = c | (torch.signbit(b).to(torch.uint8) << 3)
    return c.flatten(-2), s.view(torch.uint8)


def _values(codes, scales):
    """The numbers that codes [..., d] and scale bytes [..., d/16] stand for, fp32."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    v = table[codes.int()].unflatten(-1, (-1, 16))
    return (v * scales.view(torch.float8_e4m3fn).float()[..., None]).flatten(-2)


def _pack(k, v):
    """k, v [n, 16, d] fp32 -> tiles uint8 [n, 18 d]."""
    n, _, d = k.shape
    tiles = torch.empty(n, 18 * d, dtype=torch.uint8, device=k.device)
    ko, vo, ks, vs = _tile_offsets(d, k.device)
    for x, at, sat in ((k, ko, ks), (v, vo, vs)):
        c, s = _quantise(x)
        tiles[:, at.flatten()] = (c[..., 0::2] | (c[..., 1::2] << 4)).flatten(1)
        tiles[:, sat.flatten()] = s.flatten(1)
    return tiles


def _unpack(tiles, d):
    """tiles uint8 [..., 18 d] -> K, V [..., 16, d] fp32."""
    ko, vo, ks, vs = _tile_offsets(d, tiles.device)
    kc, vc = tiles[..., ko], tiles[..., vo]
    return (_values(torch.stack([kc & 15, kc >> 4], -1).flatten(-2), tiles[..., ks]),
            _values(torch.stack([vc & 15, vc >> 4], -1).flatten(-2), tiles[..., vs]))


# ---------------------------------------------------------------------- prepare --
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lens(case):
    """Tokens of each sequence: ragged, the last of a large batch empty."""
    lens = [max(1, case["length"] - b * case["ragged"]) for b in range(case["batch"])]
    if case["batch"] >= 16 and case["ragged"]:
        lens[-1] = 0
    return lens


def _new_lens(case):
    """Past and new tokens of each request (new < 0: the request leaves and gives its pages back)."""
    past, new = [], []
    for b in range(case["batch"]):
        p = (b * 131 + case["past"]) % (case["past"] + 1)
        n = 1
        if case["chunk"]:
            n = {0: case["chunk"], 1: 0, 7: -1}.get(b % 8, 1)
            if b % 16 == 8:
                p = 0
        past.append(p)
        new.append(n)
    return past, new


def _pages_needed(case):
    """Pages the requests hold, and the pages the step's new tokens ask for."""
    past, new = _new_lens(case)
    held = [-(-p // case["page"]) for p in past]
    want = [max(0, -(-(p + max(n, 0)) // case["page"]) - h) for p, n, h in zip(past, new, held)]
    return held, want


def prepare(case, seed):
    g = _gen(seed)
    return {"tables": _prepare_tables, "append": _prepare_append, "attend": _prepare_attend,
            "sample": _prepare_sample}[case["kind"]](case, g)


def _prepare_tables(case, g):
    past, new = _new_lens(case)
    held, want = _pages_needed(case)
    maxp = max(h + w for h, w in zip(held, want)) + 3
    pool_pages = sum(held) + case["spare"]
    pages = torch.randperm(pool_pages, generator=g, device="cuda").int()
    table = torch.full((case["batch"], maxp), -1, dtype=torch.int32, device="cuda")
    at = torch.tensor(held, device="cuda")
    first = at.cumsum(0) - at
    i = torch.arange(maxp, device="cuda")[None]
    mine = i < at[:, None]
    table[mine] = pages[(first[:, None] + i)[mine]]
    free = torch.full((pool_pages,), -1, dtype=torch.int32, device="cuda")
    free[:case["spare"]] = pages[sum(held):]
    return dict(case=case, past=torch.tensor(past, dtype=torch.int32, device="cuda"),
                new=torch.tensor(new, dtype=torch.int32, device="cuda"), table=table, free=free,
                count=torch.tensor([case["spare"]], dtype=torch.int32, device="cuda"),
                count_out=torch.zeros(1, dtype=torch.int32, device="cuda"),
                rows=sum(max(n, 0) for n in new) + 5)


def _prepare_append(case, g):
    n, hq, hkv, d, dt = case["tokens"], case["hq"], case["hkv"], case["d"], DTYPES[case["dtype"]]
    # one fused projection's output: q, k and v are column blocks of its rows
    qkv = torch.randn(n, (hq + 2 * hkv) * d, generator=g, device="cuda").to(dt)
    pages = -(-n // case["page"]) + 3
    order = torch.randperm(pages, generator=g, device="cuda")
    at = torch.arange(n, device="cuda") + 5  # the rows start inside a page
    rows = order[(at // case["page"])] * case["page"] + at % case["page"]
    st = dict(case=case, qkv=qkv, rows=rows.long(),
              pool=torch.zeros(pages, hkv, case["page"] // 16, 18 * d, dtype=torch.uint8,
                               device="cuda"),
              q_out=torch.empty(n, hq, d, dtype=dt, device="cuda"),
              qw=None, kw=None, cos=None, sin=None)
    if case["norm"]:
        st["qw"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dt)
        st["kw"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dt)
    if case["rope"]:
        freq = 1e6 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
        ang = (at + 1000).double()[:, None] * freq[None]
        ang = torch.cat([ang, ang], -1)
        st["cos"], st["sin"] = ang.cos().to(dt), ang.sin().to(dt)
    return st


def _prepare_attend(case, g):
    lens, p, d, hkv = _lens(case), case["page"], case["d"], case["hkv"]
    maxp = max(1, max(-(-n // p) for n in lens))
    pages = sum(-(-n // p) for n in lens) + 2
    tiles = pages * hkv * (p // 16)
    pool = torch.empty(tiles, 18 * d, dtype=torch.uint8, device="cuda")
    step = (1 << 24) // (16 * d)
    for at in range(0, tiles, step):
        m = min(step, tiles - at)
        pool[at:at + m] = _pack(torch.randn(m, 16, d, generator=g, device="cuda"),
                                torch.randn(m, 16, d, generator=g, device="cuda"))
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.zeros(case["batch"], maxp, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(lens):
        k = -(-n // p)
        table[b, :k] = order[at:at + k]
        at += k
    dt = DTYPES[case["dtype"]]
    mask = None
    if case["mask"] != "none":
        # left padding; with "inf" the first sequence of a batch sees nothing at all
        mask = torch.zeros(case["batch"], max(lens), dtype=dt, device="cuda")
        low = float("-inf") if case["mask"] == "inf" else torch.finfo(dt).min
        for b, n in enumerate(lens):
            pad = n if case["mask"] == "inf" and b == 0 and case["batch"] > 1 else (b * 37 % max(1, n))
            mask[b, :min(pad, n)] = low
    q = torch.randn(case["batch"], case["hq"], d, generator=g, device="cuda").to(dt)
    return dict(case=case, q=q, pool=pool.view(pages, hkv, p // 16, 18 * d), table=table,
                lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), mask=mask,
                out=torch.empty_like(q),
                lse=torch.empty(case["batch"], case["hq"], device="cuda"))


def _prepare_sample(case, g):
    b, v, mode = case["batch"], case["vocab"], case["mode"]
    logits = torch.randn(b, v, generator=g, device="cuda") * 2.5
    # a few likely tokens stand out, as they do in a language model
    best = torch.randint(v, (b, 24), generator=g, device="cuda")
    logits.scatter_add_(1, best, 9 * torch.rand(b, 24, generator=g, device="cuda"))
    r = torch.rand(5, b, generator=g, device="cuda")
    temp, top_k, top_p, min_p = 0.6 + 0.6 * r[0], None, None, None
    if mode in ("top_k", "mixed"):
        top_k = (1 + 99 * r[1]).int()
    if mode in ("top_p", "mixed"):
        top_p = 0.5 + 0.49 * r[2]
    if mode in ("min_p", "mixed"):
        min_p = 0.1 * r[3]
    if mode == "mixed":  # every filter off in some rows; some rows greedy
        i = torch.arange(b, device="cuda")
        temp = torch.where(i % 8 == 5, torch.zeros_like(temp), temp)
        top_k = torch.where(i % 3 == 0, torch.zeros_like(top_k), top_k)
        top_p = torch.where(i % 4 == 1, torch.ones_like(top_p), top_p)
        min_p = torch.where(i % 2 == 0, torch.zeros_like(min_p), min_p)
    return dict(case=case, logits=logits.to(DTYPES[case["dtype"]]), temp=temp, top_k=top_k,
                top_p=top_p, min_p=min_p, u=r[4].clone(),
                ids=torch.empty(b, dtype=torch.int64, device="cuda"),
                logp=torch.empty(b, device="cuda"))


# -------------------------------------------------------------------- plain forms --
def _plain_tables(st):
    page, b, maxp = st["case"]["page"], st["past"].numel(), st["table"].shape[1]
    past, new, free, count = st["past"].long(), st["new"].long(), st["free"].long(), st["count"].long()
    leaves = new < 0
    held = (past + page - 1) // page
    given = torch.where(leaves, held, 0)
    want = torch.where(leaves, 0, (past + new.clamp(min=0) + page - 1) // page - held)
    want = torch.where(held + want <= maxp, want, 0)
    fits = held + want >= (past + new.clamp(min=0) + page - 1) // page
    # the stack: the free pages, then the pages given back, request by request
    i = torch.arange(maxp, device=past.device)[None]
    total_given = given.sum()
    back = torch.where(leaves[:, None] & (i < held[:, None]), i + (given.cumsum(0) - given)[:, None], -1)
    at = torch.where(back >= 0, back + count, free.numel())
    stack = torch.cat([free, free.new_zeros(1)]).scatter(0, at.flatten(), st["table"].long().flatten())[:-1]
    top = count + total_given
    ends = want.cumsum(0)
    granted = fits & ((want == 0) | (ends <= top)) & ~leaves
    fresh = (i >= held[:, None]) & (i < (held + want)[:, None]) & granted[:, None]
    pick = (top - 1 - ((ends - want)[:, None] + i - held[:, None])).clamp(0, free.numel() - 1)
    table = torch.where(fresh, stack[pick], st["table"].long())
    kv = torch.where(leaves, 0, torch.where(granted, past + new, past))
    # the step's tokens, request by request
    n = new.clamp(min=0)
    cu = torch.cat([n.new_zeros(1), n.cumsum(0)])
    tok = torch.arange(st["rows"], device=past.device)
    seq = torch.searchsorted(cu[1:].contiguous(), tok, right=True)
    s = seq.clamp(max=b - 1)
    real = seq < b
    pos = past[s] + tok - cu[s]
    row = table[s, (pos // page).clamp(max=maxp - 1)] * page + pos % page
    row = torch.where(real & granted[s], row, -1)
    return dict(kv_lens=kv.int(), cu_tokens=cu.int(), seq_ids=torch.where(real, seq, -1).int(),
                positions=torch.where(real, pos, 0).int(), slot_rows=row, page_table=table.int(),
                free_pages=stack.int(), free_count=(top - (want * granted).sum()).int())


def _norm_rope(x, w, cos, sin):
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    if cos is not None:
        lo, hi = x.chunk(2, -1)
        x = x * cos.float()[:, None] + torch.cat([-hi, lo], -1) * sin.float()[:, None]
    return x


def _plain_append(st):
    c, qkv = st["case"], st["qkv"].float()
    n, hq, hkv, d, dt = c["tokens"], c["hq"], c["hkv"], c["d"], st["qkv"].dtype
    q, k, v = qkv.split([hq * d, hkv * d, hkv * d], 1)
    q = _norm_rope(q.reshape(n, hq, d), st["qw"], st["cos"], st["sin"])
    k = _norm_rope(k.reshape(n, hkv, d), st["kw"], st["cos"], st["sin"])
    v = v.reshape(n, hkv, d)
    return dict(q=q.to(dt), k=(_values(*_quantise(k / c["k_scale"])) * c["k_scale"]).to(dt),
                v=(_values(*_quantise(v / c["v_scale"])) * c["v_scale"]).to(dt))


def _plain_attend(st):
    c, q = st["case"], st["q"].float()
    b, hq, d = q.shape
    hkv = c["hkv"]
    tiles = st["pool"][st["table"].long()]  # [b, pages, hkv, tiles, 18 d]
    k, v = _unpack(tiles.transpose(1, 2).flatten(2, 3), d)
    k, v = k.flatten(2, 3) * c["k_scale"], v.flatten(2, 3) * c["v_scale"]  # [b, hkv, t, d]
    t = k.shape[2]
    s = torch.matmul(q.view(b, hkv, hq // hkv, d), k.transpose(2, 3)) * d ** -0.5
    if c["softcap"] > 0:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    seen = torch.arange(t, device=q.device)[None] < st["lens"][:, None]
    if st["mask"] is not None:
        m = torch.nn.functional.pad(st["mask"].float(), (0, max(0, t - st["mask"].shape[1])))[:, :t]
        s = s + m[:, None, None]
        seen = seen & (m > float("-inf"))
    s = torch.where(seen[:, None, None], s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp(s - top)
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p, torch.where(seen[:, None, :, None], v, 0.0)) / l.clamp(min=1e-30)
    return dict(out=o.reshape(b, hq, d).to(st["q"].dtype),
                lse=(top + torch.log(l)).reshape(b, hq))


def _plain_sample(st):
    logits, v = st["logits"].double(), st["logits"].shape[1]
    logits = torch.where(torch.isnan(logits), float("-inf"), logits)
    ls, idx = torch.sort(logits, dim=1, descending=True, stable=True)
    top = ls[:, :1]
    greedy = st["temp"] <= 0
    temp = torch.where(greedy, torch.ones_like(st["temp"]), st["temp"]).double()[:, None]
    z = torch.where(ls == top, torch.zeros_like(ls), (ls - top) / temp)
    w = torch.exp(z)
    rank = torch.arange(v, device=ls.device)[None]
    keep = torch.ones_like(w, dtype=torch.bool)
    if st["top_k"] is not None:
        k = st["top_k"].long()[:, None]
        keep = keep & ((rank < k) | (k <= 0))
    wk = torch.where(keep, w, 0.0)
    if st["top_p"] is not None:
        p, c = st["top_p"].double()[:, None], wk.cumsum(1)
        keep = keep & ((c - wk < p * c[:, -1:]) | (p >= 1) | (rank == 0))
    if st["min_p"] is not None:
        keep = keep & ((w >= st["min_p"].double()[:, None]) | (rank == 0))
    kept = torch.zeros_like(w).scatter(1, idx, torch.where(keep, w, 0.0))
    c = kept.cumsum(1)
    ids = (c <= st["u"].double()[:, None] * c[:, -1:]).sum(1).clamp(max=v - 1)
    ids = torch.where(greedy, idx[:, 0], ids)
    none = top[:, 0] == float("-inf")
    zt = (logits.gather(1, ids[:, None]) - top) / temp
    zt = torch.where(torch.isnan(zt), torch.zeros_like(zt), zt)
    logp = (zt - torch.log(w.sum(1, keepdim=True)))[:, 0].float()
    return dict(ids=torch.where(none, -1, ids), logprobs=torch.where(none, float("-inf"), logp))


# ----------------------------------------------------------- the framework's calls --
def _own_tables(st):
    from helm_b200 import _capi
    kv, cu, seq, pos, rows = _capi.build_step_tables(
        st["past"], st["new"], st["table"], st["free"], st["count"], page_size=st["case"]["page"],
        num_rows=st["rows"], free_count_out=st["count_out"])
    return dict(kv_lens=kv, cu_tokens=cu, seq_ids=seq, positions=pos, slot_rows=rows,
                page_table=st["table"], free_pages=st["free"], free_count=st["count_out"])


def _own_append(st):
    from helm_b200 import _capi
    c = st["case"]
    n, hq, hkv, d = c["tokens"], c["hq"], c["hkv"], c["d"]
    q, k, v = (x.view(n, -1, d) for x in st["qkv"].split([hq * d, hkv * d, hkv * d], 1))
    _capi.kv_append_fp4(q=q, k=k, v=v, q_out=st["q_out"], q_norm_w=st["qw"], k_norm_w=st["kw"],
                        eps=1e-6, cos=st["cos"], sin=st["sin"], pool=st["pool"],
                        slot_rows=st["rows"], page_size=c["page"], k_scale=c["k_scale"],
                        v_scale=c["v_scale"])
    kd, vd = _capi.gather_kv_rows_fp4(st["pool"], st["rows"], page_size=c["page"], dtype=q.dtype,
                                      k_scale=c["k_scale"], v_scale=c["v_scale"])
    return dict(q=st["q_out"], k=kd, v=vd)


def _own_attend(st):
    from helm_b200 import _capi
    c = st["case"]
    _capi.paged_decode_attention_fp4(
        st["q"], st["pool"], st["table"], st["lens"], num_kv_heads=c["hkv"], page_size=c["page"],
        scale=c["d"] ** -0.5, softcap=c["softcap"] or None, mask=st["mask"], k_scale=c["k_scale"],
        v_scale=c["v_scale"], out=st["out"], lse=st["lse"], max_kv_len_hint=c["length"])
    return dict(out=st["out"], lse=st["lse"])


def _own_sample(st):
    from helm_b200 import _capi
    _capi.sample_tokens(st["logits"], st["u"], temperature=st["temp"], top_k=st["top_k"],
                        top_p=st["top_p"], min_p=st["min_p"], out=st["ids"], logprobs=st["logp"])
    return dict(ids=st["ids"], logprobs=st["logp"])


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"tables": _own_tables, "append": _own_append, "attend": _own_attend,
                "sample": _own_sample}[kind](state)
    return {"tables": _plain_tables, "append": _plain_append, "attend": _plain_attend,
            "sample": _plain_sample}[kind](state)


# -------------------------------------------------------------------------- work --
def work(case):
    kind = case["kind"]
    if kind == "tables":
        past, new = _new_lens(case)
        held, want = _pages_needed(case)
        tokens = sum(max(n, 0) for n in new) + 5
        back = sum(h for h, n in zip(held, new) if n < 0)
        # lengths in and out, token rows (slot, position, request), a page entry for each page that
        # the tokens touch, the pages taken from and given back to the stack
        touched = sum(-(-(p + max(n, 0)) // case["page"]) - p // case["page"]
                      for p, n in zip(past, new) if n > 0)
        return dict(bytes=case["batch"] * 16 + tokens * 16 + touched * 4 + sum(want) * 8 + back * 8,
                    flops=0)
    if kind == "append":
        n, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
        rows = (hq + 2 * hkv) * d * 2 + hq * d * 2 + 2 * hkv * d * 9 // 16  # in, q out, pages
        back = 2 * hkv * d * 9 // 16 + 2 * hkv * d * 2                      # read back
        return dict(bytes=n * (rows + back + 8 + (4 * d if case["rope"] else 0)),
                    flops=n * ((hq + hkv) * d * (4 * case["norm"] + 3 * case["rope"]) + 6 * hkv * d))
    if kind == "attend":
        lens, d = _lens(case), case["d"]
        tokens = sum(lens)
        table = sum(-(-n // case["page"]) for n in lens) * 4
        mask = tokens * 2 if case["mask"] != "none" else 0
        return dict(bytes=tokens * case["hkv"] * d * 9 // 8 + case["batch"] * case["hq"] * (d * 4 + 4)
                    + table + mask + case["batch"] * 4,
                    flops=4 * tokens * case["hq"] * d)
    size = 4 if case["dtype"] == "fp32" else 2
    return dict(bytes=case["batch"] * (case["vocab"] * size + 32),
                flops=4 * case["batch"] * case["vocab"])


# ------------------------------------------------------------------ in 64 bits --
def _exact_block(x):
    """What a 16-value block stands for, from the definition: x float64 [..., 16]."""
    levels = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    big = x.abs().amax(-1, keepdim=True) / 6
    # e4m3: three bits after the leading one down to 2^-6, steps of 2^-9 below
    e = torch.floor(torch.log2(big.clamp(min=2.0 ** -30))).clamp(min=-6.0)
    step = torch.exp2(e - 3)
    s = (torch.round(big / step) * step).clamp(max=448.0)
    dist = (x.abs()[..., None] - s[..., None] * levels).abs()
    low = dist.amin(-1, keepdim=True)
    near = dist == low
    # of two levels at the same distance the one of even place counts
    place = torch.arange(8, device=x.device)
    pick = torch.where(near, place + 8 * (place % 2), 99).argmin(-1)
    return torch.copysign(levels[pick] * s, x)


def _exact_rows(x):
    return torch.cat([_exact_block(y.unflatten(-1, (-1, 16))).flatten(-2) for y in x.split(256)])


def _exact_append(case, st):
    n, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
    x = st["qkv"].double().view(n, hq + 2 * hkv, d)

    def turned(y, w):
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / d + 1e-6) * w.double()
        if st["cos"] is not None:
            h = d // 2
            cos, sin = st["cos"].double()[:, None], st["sin"].double()[:, None]
            y = torch.cat([y[..., :h] * cos[..., :h] - y[..., h:] * sin[..., :h],
                           y[..., h:] * cos[..., h:] + y[..., :h] * sin[..., h:]], -1)
        return y

    k = turned(x[:, hq:hq + hkv], st["kw"])
    return dict(q=turned(x[:, :hq], st["qw"]),
                k=_exact_rows(k / case["k_scale"]) * case["k_scale"],
                v=_exact_rows(x[:, hq + hkv:] / case["v_scale"]) * case["v_scale"])


def _exact_attend(case, st):
    d, hkv, page = case["d"], case["hkv"], case["page"]
    group = case["hq"] // hkv
    level = torch.tensor([(-1) ** (i >> 3) * E2M1[i & 7] for i in range(16)], dtype=torch.float64,
                         device="cuda")
    ko, vo, ks, vs = _tile_offsets(d, "cuda")
    dims = torch.arange(d, device="cuda")
    out = torch.zeros(case["batch"], case["hq"], d, dtype=torch.float64, device="cuda")
    lse = torch.full((case["batch"], case["hq"]), float("-inf"), dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lens(case)):
        if n == 0:
            continue
        pages = st["pool"][st["table"][b, :-(-n // page)].long()]
        for h in range(hkv):
            tile = pages[:, h].reshape(-1, 18 * d)

            def side(code, scale):
                byte = tile[:, code[:, dims // 2]].int()
                nib = (byte >> (4 * (dims % 2))) & 15
                s = tile[:, scale].view(torch.float8_e4m3fn).double()[..., dims // 16]
                return (level[nib] * s).reshape(-1, d)[:n]

            q = st["q"][b, h * group:(h + 1) * group].double()
            s = q @ (side(ko, ks) * case["k_scale"]).T / math.sqrt(d)
            if case["softcap"] > 0:
                s = case["softcap"] * torch.tanh(s / case["softcap"])
            if st["mask"] is not None:
                s = s + st["mask"][b, :n].double()
            if bool((s == float("-inf")).all()):
                continue
            o = torch.softmax(s, -1) @ side(vo, vs)
            out[b, h * group:(h + 1) * group] = o * case["v_scale"]
            lse[b, h * group:(h + 1) * group] = torch.logsumexp(s, -1)
    return dict(out=out, lse=lse)


def _exact_sample(case, st):
    ids, logp = [], []
    for i, row in enumerate(st["logits"].double()):
        t = float(st["temp"][i])
        z = row / (t if t > 0 else 1.0)
        total = torch.logsumexp(z, 0)
        order = torch.sort(row, descending=True, stable=True).indices
        if t > 0:
            if st["top_k"] is not None and int(st["top_k"][i]) > 0:
                order = order[:int(st["top_k"][i])]
            if st["top_p"] is not None and float(st["top_p"][i]) < 1:
                mass = torch.softmax(z[order], 0).cumsum(0)
                short = int((mass < float(st["top_p"][i])).sum())
                order = order[:short + 1]
            if st["min_p"] is not None and float(st["min_p"][i]) > 0:
                order = order[torch.exp(z[order] - z[order[0]]) >= float(st["min_p"][i])]
            kept = order.sort().values
            mass = torch.softmax(z[kept], 0).cumsum(0)
            ids.append(int(kept[min(len(kept) - 1, int((mass <= float(st["u"][i])).sum()))]))
        else:
            ids.append(int(order[0]))
        logp.append(z[ids[-1]] - total)
    return dict(ids=torch.tensor(ids), logprobs=torch.stack(logp))


def exact(case, seed):
    if case["kind"] == "tables":
        return None  # whole numbers: nothing is rounded
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](
        case, st)
