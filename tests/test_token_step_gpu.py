"""TPDecodeModel over 4-bit pages when pages run out, sequences idle, and contexts are
filled in (GPU)."""
import pytest
import torch

from helm_b200 import _capi
from helm_b200.runtime.sampling import SamplingParams
from helm_b200.runtime.tp_decode import TPDecodeModel, synthetic_shard
from test_serving_step_gpu import ARCH, dev  # noqa: F401

pytestmark = pytest.mark.gpu


def _model(dev, **kw):  # noqa: F811
    w = synthetic_shard(ARCH, 0, 1, torch.bfloat16, dev, seed=2, std=0.06)
    tp = TPDecodeModel(w, batch=2, max_len=64, page_size=16, kv_format="fp4", **kw)
    tp.ids.copy_(torch.tensor([[5], [6]]))
    return tp


@pytest.mark.parametrize("how", ["step", "replay", "forced", "sampled"])
def test_a_refused_sequence_keeps_its_token(dev, how):  # noqa: F811
    """Sequence 1 finds no page for its 17th token, waits, and goes on as if it had not."""
    kw = {}
    if how == "sampled":
        kw["sampling"] = SamplingParams(temperature=0.0)
    tp, free = _model(dev, num_pages=3, **kw), _model(dev, **kw)
    if how == "replay":
        tp.capture()

    def step(model):
        if how == "replay" and model is tp:
            model.replay()
        elif how == "forced":
            model.step(torch.tensor([[3], [int(model.lens[1]) % 500 + 1]], device=dev))
        else:
            model.step()

    want = []
    for _ in range(40):
        step(free)
        want.append((free.full_logits()[1].cpu(), int(free.ids[1])))
    for t in range(16):
        step(tp)
        assert int(tp.ids[1]) == want[t][1]
    for _ in range(16):   # sequence 0 has the third page
        step(tp)
        assert tp.lens[1].item() == 16 and int(tp.ids[1]) == want[15][1]
    assert tp.lens[0].item() == 32 and _capi.device_status(dev) == _capi.DEV_NO_PAGES
    tp.set_step([-1, 1])   # sequence 0 leaves, sequence 1 gets a page of its own
    for t in range(16, 32):
        step(tp)
        assert torch.equal(tp.full_logits()[1].cpu(), want[t][0]) and int(tp.ids[1]) == want[t][1]
    assert tp.lens.tolist() == [0, 32] and _capi.device_status(dev) == 0
    tp.close()
    free.close()


def test_an_idle_sequence_keeps_its_token_unless_told(dev):  # noqa: F811
    tp = _model(dev)
    tp.set_step([1, 0])
    tp.step()
    assert int(tp.ids[1]) == 6
    tp.step(torch.tensor([[8], [9]]))   # (what it is to start with may be given)
    assert tp.ids.view(-1).tolist() == [8, 9] and tp.lens.tolist() == [2, 0]
    tp.close()


def test_fill_kv_and_the_device_status(dev):  # noqa: F811
    """A refused context changes nothing; an old status neither stops fill_kv nor is lost."""
    tp = _model(dev, num_pages=5)
    for _ in range(49):
        tp.step()
    assert tp.lens.sum().item() == 80
    before = [t.clone() for t in (tp.lens, tp.table, tp.free_pages, tp.free_count, *tp.pools)]
    with pytest.raises(ValueError):
        tp.fill_kv(40)   # 6 pages
    after = (tp.lens, tp.table, tp.free_pages, tp.free_count, *tp.pools)
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    tp.fill_kv(20)       # fits, whatever happened before
    assert tp.lens.tolist() == [20, 20] and tp.free_count.item() == 1
    assert _capi.device_status(dev) == _capi.DEV_NO_PAGES
    tp.close()
