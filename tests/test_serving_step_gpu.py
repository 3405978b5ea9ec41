"""The 4-bit cache, the step tables and the sampler as the decode models use them:
a run of steps of TPDecodeModel(kv_format="fp4", sampling=...), and sampling in
DecodeLoop and GraphDecoder (GPU).

The 4-bit model is compared with a float64 forward of each token over the cache
that the model itself wrote (read from its pages): what is left are bf16 roundings
of one token's activations, the same as in the 16-bit model, so the bar is the
16-bit model's distance from a float64 forward over its cache.  (A float64 run that
quantises its own K and V would not do: activations that differ by a bf16 rounding
put a few percent of the values on the other side of a border between codes.)
"""
import numpy as np
import pytest
import torch

from helm_b200 import _capi
from helm_b200.runtime.decode_loop import DecodeLoop
from helm_b200.runtime.graph_decode import GraphDecoder
from helm_b200.runtime.kv_offload import KVOffloadConfig, KVOffloadManager
from helm_b200.runtime.sampling import SamplingParams, TokenSampler
from helm_b200.runtime.tp_decode import TPDecodeModel, synthetic_shard
from helm_b200.synthetic import build_model, make_config
from oracle import fp4, serving

pytestmark = pytest.mark.gpu

ARCH = dict(hidden=256, layers=2, q_heads=4, kv_heads=2, head_dim=64, intermediate=512, vocab=512,
            qk_norm=True, theta=1e6)


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("CUDA device required")
    return torch.device("cuda:0")


class Exact:
    """The decode step of one token in float64 over K, V read from the model's cache."""

    def __init__(self, w):
        self.w = w
        self.d = lambda t: t.double().cpu().numpy()

    def _rms(self, x, weight, eps):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * self.d(weight)

    def step(self, cache, token):
        """cache: per layer K, V [tokens, Hkv, D], this token's rows among them.  Returns the
        logits and, per layer, how far the token's own K and V are from the cached ones
        relative to their blocks' largest values."""
        w, d, far = self.w, self.d, []
        D, pos = w.head_dim, cache[0][0].shape[0] - 1
        h = d(w.embed[token])
        ang = pos * w.theta ** (-np.arange(0, D, 2) / D)
        cos, sin = np.concatenate([np.cos(ang)] * 2), np.concatenate([np.sin(ang)] * 2)

        def turn(x):
            return x * cos + np.concatenate([-x[:, D // 2:], x[:, :D // 2]], -1) * sin

        for l, (ks, vs) in zip(w.layers, cache):
            qkv = (d(l.wqkv) @ self._rms(h, l.ln1, l.eps1)).reshape(-1, D)
            q, k, v = qkv[:w.hq], qkv[w.hq:w.hq + w.hkv], qkv[w.hq + w.hkv:]
            if l.q_norm is not None:
                q, k = self._rms(q, l.q_norm, l.qk_eps), self._rms(k, l.k_norm, l.qk_eps)
            q, k = turn(q), turn(k)
            for x, c in ((k, ks[-1]), (v, vs[-1])):
                top = np.abs(x.reshape(-1, 16)).max(-1, keepdims=True)
                far.append((np.abs(c - x).reshape(-1, 16) / top).max())
            o, _, _ = fp4.attention(q, ks, vs, D ** -0.5)
            h = h + d(l.wo) @ o.reshape(-1)
            x = self._rms(h, l.ln2, l.eps2)
            g, u = d(l.wg) @ x, d(l.wu) @ x
            h = h + d(l.wd) @ (g / (1 + np.exp(-g)) * u)
        return d(w.lm_head) @ self._rms(h, w.final_norm, w.final_eps), max(far)


def _cached(tp, b, n):
    """Per layer K, V float64 [n, Hkv, D] of sequence b, from the model's pages."""
    out = []
    for l in range(tp.L):
        table = (tp.table if tp.fp4 else tp.tables[l])[b].tolist()
        rows = [table[t // tp.P] * tp.P + t % tp.P for t in range(n)]
        if tp.fp4:
            out.append(fp4.read_rows(tp.pools[l].cpu().numpy(), rows, tp.P))
        else:
            x = tp.pool.double().cpu().numpy()
            out.append([np.stack([x[r // tp.P, i, :, r % tp.P] for r in rows]) for i in (0, 1)])
    return out


def _errors(dev, kv_format, tokens):
    w = synthetic_shard(ARCH, 0, 1, torch.bfloat16, dev, seed=1, std=0.06)
    tp = TPDecodeModel(w, batch=tokens.shape[0], max_len=80, page_size=16, kv_format=kv_format)
    exact, err, far = Exact(w), [], 0.0
    for t in range(tokens.shape[1]):
        tp.ids.copy_(tokens[:, t:t + 1])
        tp.step()
        got = tp.full_logits().double().cpu().numpy()
        for b in range(tokens.shape[0]):
            want, f = exact.step(_cached(tp, b, t + 1), int(tokens[b, t]))
            err.append(np.abs(got[b] - want))
            far = max(far, f)
    assert _capi.device_status(dev) == 0
    tp.close()
    return np.stack(err), far


def test_the_4_bit_model_is_as_exact_as_the_16_bit_one(dev):
    tokens = torch.randint(0, ARCH["vocab"], (2, 40), generator=torch.Generator().manual_seed(3))
    (e16, far16), (e4, far4) = _errors(dev, "model", tokens), _errors(dev, "fp4", tokens)
    assert e4.max() <= 1.5 * e16.max() + 2e-2, (e4.max(), e16.max())
    assert e4.mean() <= 1.25 * e16.mean() + 1e-3, (e4.mean(), e16.mean())
    # the cached values: half of the widest gap between levels (1 of 6 scales' worth, the scale
    # itself off by 2^-4 at most) beyond what the 16-bit model's are off
    assert far4 <= (1 + 2.0 ** -4) / 6 + far16 * 1.5 + 1e-3, (far4, far16)


def _serve(tp, dev, plan, replay):
    """Runs the plan of steps; what each sequence saw, and the logits of every step."""
    rows = []
    if replay:
        tp.capture()
    for new in plan:
        tp.set_step(new)
        (tp.replay if replay else tp.step)()
        rows.append((tp.lens.tolist(), tp.ids.view(-1).tolist(), tp.full_logits().cpu(),
                     tp.table.tolist(), tp.free_count.item()))
    assert _capi.device_status(dev) == 0
    return rows


def test_requests_come_and_go_over_shared_pages(dev):
    """Three sequences share 9 pages of 16 tokens: steps with idle and leaving ones.  Pages and
    lengths are the host's, a sequence's logits do not depend on the others or on the pages it
    got, and the replayed run is the eager one bit for bit."""
    plan = [[1, 1, 0]] * 20 + [[1, 0, 1]] * 15 + [[1, -1, 1]] + [[1, 0, 1]] * 4 + [[1, 1, 1]] * 24
    w = synthetic_shard(ARCH, 0, 1, torch.bfloat16, dev, seed=2, std=0.06)

    def model(**kw):
        tp = TPDecodeModel(w, batch=3, max_len=96, page_size=16, kv_format="fp4", num_pages=9, **kw)
        tp.ids.copy_(torch.tensor([[5], [6], [7]]))
        return tp

    tp = model()
    eager = _serve(tp, dev, plan, False)
    tp.close()
    tp = model()
    replayed = _serve(tp, dev, plan, True)
    tp.close()
    for a, b in zip(eager, replayed):
        assert a[:2] == b[:2] and a[3:] == b[3:]
        assert torch.equal(a[2], b[2])
    # the pages and lengths, restated on the host
    lens, table, free, count = [0, 0, 0], [[-1] * 6] * 3, list(range(8, -1, -1)), 9
    for new, (got_lens, _, _, got_table, got_count) in zip(plan, eager):
        r = serving.step_tables(lens, new, table, free, count, 16, 3)
        lens, table, free, count = r["kv_lens"], r["page_table"], r["free_pages"], r["free_count"]
        assert not r["refused"]
        assert (got_lens, got_table, got_count) == (lens, table, count)
    # sequence 1 alone, with pages of its own: the same tokens up to its leaving
    alone = TPDecodeModel(w, batch=3, max_len=96, page_size=16, kv_format="fp4")
    alone.ids.copy_(torch.tensor([[9], [6], [9]]))
    alone.set_step([0, 1, 0])
    for t in range(20):
        alone.step()
        assert torch.equal(alone.full_logits()[1].cpu(), eager[t][2][1])
    alone.close()


def test_fill_kv_starts_over(dev):
    w = synthetic_shard(ARCH, 0, 1, torch.bfloat16, dev, seed=2)
    tp = TPDecodeModel(w, batch=2, max_len=64, page_size=16, kv_format="fp4")
    for length in (40, 17, 0, 63):
        tp.fill_kv(length)
        held = 2 * -(-length // 16)
        assert tp.lens.tolist() == [length] * 2 and tp.free_count.item() == 8 - held
        pages = tp.table[:, :held // 2].flatten().tolist() + tp.free_pages[:8 - held].tolist()
        assert sorted(pages) == list(range(8))
    tp.step()
    assert tp.lens.tolist() == [64, 64] and _capi.device_status(dev) == 0
    tp.close()


def test_running_out_of_pages_is_reported(dev):
    w = synthetic_shard(ARCH, 0, 1, torch.bfloat16, dev, seed=2)
    tp = TPDecodeModel(w, batch=2, max_len=64, page_size=16, kv_format="fp4", num_pages=3)
    for _ in range(32):
        tp.step()
    assert tp.lens.tolist() == [32, 16] and tp.free_count.item() == 0
    assert _capi.device_status(dev) == _capi.DEV_NO_PAGES
    tp.set_step([1, -1])   # the second leaves: its page serves the first
    tp.step()
    assert tp.lens.tolist() == [33, 0] and _capi.device_status(dev) == 0
    with pytest.raises(ValueError):
        tp.set_step([1, 2])
    with pytest.raises(ValueError):
        tp.fill_kv(63)
    tp.close()
    with pytest.raises(ValueError):
        TPDecodeModel(w, batch=1, max_len=64, kv_format="int3")
    with pytest.raises(ValueError):
        TPDecodeModel(w, batch=1, max_len=64, num_pages=3)


@pytest.mark.parametrize("kv_format", ["model", "fp4"])
def test_sampled_decode(dev, kv_format):
    """Every step's token is the oracle's draw from the step's logits; replays draw anew."""
    params = SamplingParams(temperature=[0.8, 0.0], top_k=[0, 5], top_p=0.9, min_p=0.01, seed=11)
    w = synthetic_shard(ARCH, 0, 1, torch.bfloat16, dev, seed=4, std=0.06)
    tp = TPDecodeModel(w, batch=2, max_len=64, page_size=16, kv_format=kv_format, sampling=params)
    u = torch.rand(TokenSampler.ROWS, 2, generator=torch.Generator().manual_seed(11))
    for step in range(12):
        if step == 4:
            tp.capture()
        (tp.step if step < 4 else tp.replay)()
        logits = tp.full_logits().double().cpu().numpy()
        for b in range(2):
            tok, lp = serving.sample(logits[b], float(u[step, b]), float(np.float32([0.8, 0.0][b])),
                                     [0, 5][b], float(np.float32(0.9)), float(np.float32(0.01)))
            assert int(tp.ids[b]) == tok
            assert abs(float(tp.sampler.logprobs[b]) - lp) <= 1e-5
    assert _capi.device_status(dev) == 0
    tp.close()


def test_sampling_in_the_loops(dev):
    """DecodeLoop and GraphDecoder draw from the same uniforms; every token is the oracle's draw."""
    cfg = make_config("tiny", family="qwen3", layers=2, hidden=512, q_heads=8, kv_heads=4,
                      head_dim=128, intermediate=1024, vocab=512)
    model = build_model(cfg, seed=0, std=0.05, dtype=torch.bfloat16, device="cuda")
    prompt = torch.randint(0, 512, (2, 48), generator=torch.Generator().manual_seed(0)).cuda()
    params = SamplingParams(temperature=0.9, top_k=40, top_p=0.95, seed=5)
    u = torch.rand(TokenSampler.ROWS, 2, generator=torch.Generator().manual_seed(5))
    n = 10
    for kind in ("loop", "graph"):
        mgr = KVOffloadManager(model, KVOffloadConfig.from_model(model, page_size=16), batch_size=2)
        try:
            if kind == "loop":
                toks, logits = DecodeLoop(model, mgr).generate(prompt, n, keep_logits=True,
                                                               sampling=params)
            else:
                toks, logits = GraphDecoder(model, mgr, max_len=48 + n).generate(
                    prompt, n, keep_logits=True, sampling=params)
        finally:
            mgr.restore()
        for s in range(n):
            for b in range(2):
                want, _ = serving.sample(logits[s][b].double().cpu().numpy(), float(u[s, b]),
                                         float(np.float32(0.9)), 40, float(np.float32(0.95)))
                assert int(toks[b, s]) == want, (kind, s, b)
    mgr = KVOffloadManager(model, KVOffloadConfig.from_model(model, page_size=16), batch_size=2)
    try:
        greedy = DecodeLoop(model, mgr).generate(prompt, 4)
        zero = DecodeLoop(model, mgr).generate(prompt, 4, sampling=SamplingParams(temperature=0.0))
    finally:
        mgr.restore()
    assert torch.equal(greedy, zero)


def test_sampler_refills_and_refuses(dev):
    s = TokenSampler(SamplingParams(seed=3), 1, dev)
    logits = torch.zeros(1, 50000, device=dev)
    gen = torch.Generator().manual_seed(3)
    u = torch.cat([torch.rand(TokenSampler.ROWS, 1, generator=gen) for _ in range(2)])
    for step in range(TokenSampler.ROWS + 3):
        s.tick()
        tok = int(s(logits)) if step in (0, 1, TokenSampler.ROWS, TokenSampler.ROWS + 2) else s(logits)
        if not torch.is_tensor(tok):
            assert tok == serving.sample(np.zeros(50000), float(u[step]))[0]
    s.tick()
    assert int(s(torch.full((1, 9), float("-inf"), device=dev))) == 0
    for bad in (dict(temperature=-1.0), dict(top_p=1.5), dict(min_p=-0.1), dict(top_k=[1, 2])):
        with pytest.raises(ValueError):
            TokenSampler(SamplingParams(**bad), 1, dev)
