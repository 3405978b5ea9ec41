"""Calls on a stream of their own while the current one is still busy (GPU): what a call
allocates is not memory that queued work on the current stream still reads."""
import pytest
import torch

from helm_b200 import _capi

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("CUDA device required")
    return torch.device("cuda:0")


def _attention(dev):
    g = torch.Generator().manual_seed(1)
    pool = _capi.fp4_pool(40, 2, 16, 128, dev)
    x = torch.randn(600, 2, 128, generator=g).to(BF16).to(dev)
    _capi.kv_append_fp4(k=x, v=x, pool=pool, slot_rows=torch.arange(600, device=dev), page_size=16)
    q = torch.randn(1, 8, 128, generator=g).to(BF16).to(dev)
    table = torch.arange(40, dtype=torch.int32, device=dev).view(1, -1)
    lens = torch.tensor([600], dtype=torch.int32, device=dev)

    def call(stream=None):
        return [_capi.paged_decode_attention_fp4(q, pool, table, lens, num_kv_heads=2, page_size=16,
                                                 scale=0.09, stream=stream)[0]]
    return call


def _gather(dev):
    pool = torch.randint(0, 127, (40, 2, 1, 18 * 128), dtype=torch.uint8, device=dev)
    rows = torch.arange(600, device=dev)
    return lambda stream=None: _capi.gather_kv_rows_fp4(pool, rows, page_size=16, dtype=BF16,
                                                        stream=stream)


def _tables(dev):
    b = 2000
    i32 = dict(dtype=torch.int32, device=dev)
    past, new = torch.arange(b, **i32), torch.ones(b, **i32)
    # (the call writes its table, stack and count: a set for each)
    sets = [(torch.arange(b * 130, **i32).view(b, 130), torch.arange(b, **i32),
             torch.full((1,), b, **i32)) for _ in range(2)]

    def call(stream=None):
        table, free, count = sets.pop()
        return _capi.build_step_tables(past, new, table, free, count, page_size=16, num_rows=b,
                                       stream=stream)
    return call


def _sample(dev):
    x = torch.randn(3000, 400, generator=torch.Generator().manual_seed(3)).to(dev)
    u = torch.rand(3000, generator=torch.Generator().manual_seed(4)).to(dev)
    return lambda stream=None: [_capi.sample_tokens(x, u, stream=stream)]


@pytest.mark.parametrize("make", [_attention, _gather, _tables, _sample])
def test_a_call_beside_a_busy_stream(dev, make):
    call = make(dev)
    want = [t.clone() for t in call()]
    side = torch.cuda.Stream(dev)
    torch.cuda.synchronize(dev)
    torch.cuda.empty_cache()
    # blocks of every size that the call may ask for, freed while their readers are queued
    sizes = [2 ** i for i in range(9, 28)]
    sizes.append(int(_capi.lib().helm_paged_decode_fp4_workspace_bytes(1, 8, 2, 128)))
    blocks = [torch.full((n,), 7, dtype=torch.uint8, device=dev) for n in sizes for _ in range(2)]
    for b in blocks[:1] + blocks[-1:]:   # (loading their kernels would wait for the device)
        b.amin(), b.amax()
    torch.cuda.synchronize(dev)
    torch.cuda._sleep(400_000_000)   # ~0.2 s
    seen = [(b.amin(), b.amax()) for b in blocks]   # (no scratch of their size)
    del blocks
    got = call(stream=side)
    side.synchronize()
    torch.cuda.synchronize(dev)
    assert all(int(lo) == int(hi) == 7 for lo, hi in seen)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
