"""Step tables on the GPU against the host restatement, request by request: every
output is a whole number and has to be equal."""
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


def _case(seed, batch, page, maxp, most_past, most_new, spare, capacity=None):
    g = np.random.default_rng(seed)
    past = g.integers(0, most_past + 1, batch)
    new = g.integers(-1, most_new + 1, batch)
    held = -(-past // page)
    n = int(held.sum()) + spare
    ids = g.permutation(n).astype(np.int32)
    table = np.full((batch, maxp), -7, np.int32)
    at = 0
    for b in range(batch):
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    cap = n if capacity is None else capacity
    free = np.full(cap, -9, np.int32)
    free[:spare] = ids[at:]
    return past, new, table, free, spare


def _run(dev, past, new, table, free, count, page, num_rows, **kw):
    t = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    past, table, free, count = t(past), t(table), t(free), t([count])
    kv, cu, seq, pos, rows = _capi.build_step_tables(past, t(new), table, free, count,
                                                     page_size=page, num_rows=num_rows, **kw)
    return dict(kv_lens=kv, cu_tokens=cu, seq_ids=seq, positions=pos, slot_rows=rows,
                page_table=table, free_pages=free, free_count=count)


def _check(dev, past, new, table, free, count, page, num_rows):
    want = serving.step_tables(past.tolist(), new.tolist(), table.tolist(), free.tolist(), count,
                               page, num_rows)
    got = _run(dev, past, new, table, free, count, page, num_rows)
    status = _capi.device_status(dev)
    assert status == (_capi.DEV_NO_PAGES if want.pop("refused") else 0)
    want["free_count"] = [want["free_count"]]
    for name, w in want.items():
        assert got[name].cpu().tolist() == w, name


@pytest.mark.parametrize("batch,page,most_past,most_new,spare", [
    (1, 16, 0, 1, 1), (1, 16, 16, 1, 3), (16, 16, 100, 1, 40), (37, 64, 300, 90, 200),
    (300, 16, 64, 3, 400), (513, 32, 100, 40, 1500), (2000, 16, 50, 2, 3000)])
def test_against_the_host(dev, batch, page, most_past, most_new, spare):
    maxp = -(-(most_past + most_new) // page) + 2
    past, new, table, free, count = _case(batch + page, batch, page, maxp, most_past, most_new, spare)
    _check(dev, past, new, table, free, count, page, int(np.maximum(new, 0).sum()) + 3)


def test_many_tokens_run_over_several_ctas(dev):
    past, new, table, free, count = _case(3, 40, 16, 120, 500, 1300, 4000)
    total = int(np.maximum(new, 0).sum())
    assert total > 4 * 2048
    _check(dev, past, new, table, free, count, 16, total)


@pytest.mark.parametrize("spare", [0, 1, 7, 20])
def test_too_few_pages(dev, spare):
    past, new, table, free, count = _case(5, 30, 16, 10, 60, 40, spare)
    _check(dev, past, new, table, free, count, 16, int(np.maximum(new, 0).sum()) + 1)


def test_rows_of_the_table_too_short(dev):
    past, new, table, free, count = _case(7, 30, 16, 4, 64, 40, 100)
    _check(dev, past, new, table, free, count, 16, int(np.maximum(new, 0).sum()))


def test_stack_too_small_for_the_pages_given_back(dev):
    past, new, table, free, count = _case(9, 30, 16, 12, 120, 1, 5, capacity=9)
    new[:] = -1
    got = _run(dev, past, new, table, free, count, 16, 2)
    assert _capi.device_status(dev) == _capi.DEV_NO_PAGES
    assert got["free_count"].item() == 9 and (got["slot_rows"] == -1).all()
    assert got["free_pages"][:5].tolist() == free[:5].tolist()


def test_fewer_rows_than_tokens_and_none(dev):
    past, new, table, free, count = _case(11, 8, 16, 8, 30, 9, 60)
    _check(dev, past, new, table, free, count, 16, 5)
    _check(dev, past, new, table, free, count, 16, 0)


def test_empty_stack(dev):
    past, new = np.array([3, 16, 0]), np.array([1, 1, 0])
    table = np.array([[5, -7], [6, -7], [-7, -7]], np.int32)
    _check(dev, past, new, table, np.zeros(0, np.int32), 0, 16, 4)


@pytest.mark.parametrize("num_rows", [8, 20001])
def test_absurd_lengths_are_refused_in_bounds(dev, num_rows):
    most = 2 ** 31 - 1
    got = _run(dev, [0, 5, most, 1], [most, most, most, 1],
               np.array([[0, 1], [2, 3], [4, 5], [6, 7]], np.int32), [8, 9], 2, 16, num_rows)
    assert _capi.device_status(dev) == _capi.DEV_NO_PAGES
    assert got["kv_lens"].tolist()[:3] == [0, 5, most]
    assert got["cu_tokens"].tolist() == [0, most, most, most, most]
    assert got["seq_ids"].tolist() == [0] * num_rows
    assert got["slot_rows"].tolist() == [-1] * num_rows
    assert got["free_count"].tolist() == [2]


def test_all_leave_and_all_idle(dev):
    past, new, table, free, count = _case(13, 20, 16, 8, 100, 3, 4)
    _check(dev, past, np.full_like(new, -1), table, free, count, 16, 4)
    _check(dev, past, np.zeros_like(new), table, free, count, 16, 4)


def test_steps_in_place_and_captured(dev):
    """Lengths and the stack's count updated in place, the step replayed as a graph."""
    batch, page, maxp = 6, 16, 9
    lens = torch.tensor([15, 0, 31, 47, 16, 100], dtype=torch.int32, device=dev)
    host = [15, 0, 31, 47, 16, 100]
    new = torch.ones(batch, dtype=torch.int32, device=dev)
    ids = list(range(100))
    table = np.zeros((batch, maxp), np.int64)
    at = 0
    for b, n in enumerate(host):
        for i in range(-(-n // page)):
            table[b, i] = ids[at]
            at += 1
    count = 100 - at
    free = ids[at:] + [0] * at
    t = torch.tensor(table, dtype=torch.int32, device=dev)
    f = torch.tensor(free, dtype=torch.int32, device=dev)
    c = torch.tensor([count], dtype=torch.int32, device=dev)
    out = dict(cu_tokens=torch.empty(batch + 1, dtype=torch.int32, device=dev),
               slot_rows=torch.empty(batch, dtype=torch.int64, device=dev))

    def step():
        _capi.build_step_tables(lens, new, t, f, c, page_size=page, num_rows=batch, kv_lens=lens,
                                **out)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    tab = table.tolist()
    for i in range(20):
        n = [1] * batch
        if i == 7:
            n[5] = -1
        if i > 7:
            n[5] = 0
        new.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        r = serving.step_tables(host, n, tab, free, count, page, batch)
        host, tab, free, count = r["kv_lens"], r["page_table"], r["free_pages"], r["free_count"]
        torch.cuda.synchronize(dev)
        assert lens.tolist() == host and c.item() == count
        assert out["slot_rows"].tolist() == r["slot_rows"]
        assert t.tolist() == tab and f.tolist() == free
    assert _capi.device_status(dev) == 0


def test_wrapper_refusals(dev):
    i = torch.zeros(4, dtype=torch.int32, device=dev)
    tab = torch.zeros(4, 3, dtype=torch.int32, device=dev)
    call = _capi.build_step_tables
    for bad in (lambda: call(i.long(), i, tab, i, i[:1], page_size=16, num_rows=4),
                lambda: call(i, i[:3], tab, i, i[:1], page_size=16, num_rows=4),
                lambda: call(i, i, tab[:3], i, i[:1], page_size=16, num_rows=4),
                lambda: call(i, i, tab, i, i, page_size=16, num_rows=4),
                lambda: call(i, i, tab, i.cpu(), i[:1], page_size=16, num_rows=4),
                lambda: call(i, i, tab, i, i[:1], page_size=0, num_rows=4),
                lambda: call(i, i, tab, i, i[:1], page_size=16, num_rows=4,
                             slot_rows=torch.empty(3, dtype=torch.int64, device=dev))):
        with pytest.raises(_capi.HelmError):
            bad()
