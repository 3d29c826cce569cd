"""The hook that lets the pool's slots follow a cache layer's rows (host logic, CPU)."""
import copy
import pickle

import torch

from nested_ssm_b200 import hf


class Layer:
    def __init__(self):
        self.rows = torch.arange(4)

    def reorder_cache(self, beam_idx):
        self.rows = self.rows[beam_idx]


def _state(calls, monkeypatch):
    def reorder(buffers, slots, parents):
        calls.append((buffers, slots.tolist(), parents.tolist()))
        return slots[parents]

    monkeypatch.setattr(hf, "reorder_slots", reorder)
    return {"pool": "pool", "slots": torch.tensor([3, 1, 0, 2]), "draft": None}


def test_rows_and_slots_are_reordered_once_per_call(monkeypatch):
    calls = []
    layer, st = Layer(), _state(calls, monkeypatch)
    hf._follow_beams(layer, st)
    hf._follow_beams(layer, st)           # a second prefill on the same cache
    layer.reorder_cache(torch.tensor([1, 1, 2, 0]))
    assert layer.rows.tolist() == [1, 1, 2, 0] and st["slots"].tolist() == [1, 1, 0, 3]
    assert calls == [("pool", [3, 1, 0, 2], [1, 1, 2, 0])]


def test_a_deep_copy_reorders_its_own_rows(monkeypatch):
    layer, st = Layer(), _state([], monkeypatch)
    hf._follow_beams(layer, st)
    other = copy.deepcopy([layer])[0]
    other.reorder_cache(torch.tensor([3, 2, 1, 0]))
    assert other.rows.tolist() == [3, 2, 1, 0] and layer.rows.tolist() == [0, 1, 2, 3]
    assert other.reorder_cache.st is st


def test_a_layer_without_rows_to_reorder_is_left_alone():
    class Plain:
        pass

    layer = Plain()
    hf._follow_beams(layer, {})
    assert not hasattr(layer, "reorder_cache")


def test_a_layer_goes_with_its_last_reference(monkeypatch):
    import gc
    import weakref
    layer, st = Layer(), _state([], monkeypatch)
    hf._follow_beams(layer, st)
    gc.disable()
    try:
        gone = weakref.ref(layer)
        del layer
        assert gone() is None
    finally:
        gc.enable()


def test_a_shallow_copy_reorders_its_own_rows(monkeypatch):
    layer, st = Layer(), _state([], monkeypatch)
    hf._follow_beams(layer, st)
    other = copy.copy(layer)
    other.reorder_cache(torch.tensor([3, 2, 1, 0]))
    assert other.rows.tolist() == [3, 2, 1, 0] and layer.rows.tolist() == [0, 1, 2, 3]
    assert st["slots"].tolist() == [2, 0, 1, 3]


def test_a_layer_can_be_pickled_and_saved(monkeypatch, tmp_path):
    """What is read back is a layer of the plain class: the pool stays with the model."""
    layer, st = Layer(), _state([], monkeypatch)
    hf._follow_beams(layer, st)
    cache = {"layers": [layer, layer]}
    torch.save(cache, tmp_path / "cache.pt")
    for got in (pickle.loads(pickle.dumps(cache)), torch.load(tmp_path / "cache.pt", weights_only=False)):
        first, second = got["layers"]
        assert first is second and type(first) is Layer and first.rows.tolist() == [0, 1, 2, 3]
        first.reorder_cache(torch.tensor([1, 0, 3, 2]))
        assert first.rows.tolist() == [1, 0, 3, 2]
    assert st["slots"].tolist() == [3, 1, 0, 2] and isinstance(layer, Layer) and layer.reorder_cache.st is st


def test_an_older_cache_leaves_the_pool_to_the_newer(monkeypatch):
    """A mixer has one pool: after another cache's prefill it holds that cache's states."""
    calls = []
    old, new, st = Layer(), Layer(), _state(calls, monkeypatch)
    hf._follow_beams(old, st)
    kept = copy.deepcopy(old)
    hf._follow_beams(new, st)
    for layer in (old, kept):
        layer.reorder_cache(torch.tensor([1, 0]))      # fewer rows than the pool's, too
        assert layer.rows.tolist() == [1, 0]
    assert not calls and st["slots"].tolist() == [3, 1, 0, 2]
    copy.deepcopy(new).reorder_cache(torch.tensor([1, 1, 2, 0]))
    assert len(calls) == 1 and st["slots"].tolist() == [1, 1, 0, 3]


def test_moves_of_the_draft_report_to_the_pool(monkeypatch):
    """The draft's buffers are described once and share the pool's status word."""
    made, calls = [], []

    class Buffers:
        def __init__(self, tensors):
            self.tensors, self.status = tensors, "its own"
            made.append(self)

    class Pool:
        status = "the pool's"

    monkeypatch.setattr(hf, "StateBuffers", Buffers)
    layer, st = Layer(), _state(calls, monkeypatch)
    st["pool"], st["draft"] = Pool(), torch.zeros(4, 2)
    hf._follow_beams(layer, st)
    for _ in range(3):
        layer.reorder_cache(torch.tensor([1, 0, 2, 3]))
    assert len(made) == 1 and made[0].tensors[0] is st["draft"] and made[0].status is Pool.status
    assert [c[0] for c in calls] == [made[0], st["pool"]] * 3
    st["draft"] = torch.zeros(4, 2)          # a larger batch's prefill makes another
    layer.reorder_cache(torch.tensor([1, 0, 2, 3]))
    assert len(made) == 2 and made[1].tensors[0] is st["draft"]
