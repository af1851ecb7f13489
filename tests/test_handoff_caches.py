"""The prefill hand-off on the CPU: which caches get the queries' weights with the anchors."""
from types import SimpleNamespace

import pytest
import torch

pytest.importorskip("transformers")


def _packed(P=6):
    rows = torch.zeros(1, 2, P, 32)
    ones = torch.ones(1, 2, P, dtype=torch.int32)
    p = SimpleNamespace(k_packed=rows, v_packed=rows, counts=ones, timestamps=ones, anchor_counts=ones.sum(-1, dtype=torch.int32))
    p.trimmed = lambda: p
    return p


class _OtherCache:
    """A cache of the caller's own, with attributes that mean something else here."""
    exact_window_size = 4
    budget = 3
    observe = None
    got = None

    def initialize_from_prefill(self, layer_idx, k_packed, v_packed, counts, timestamps, k_exact, v_exact, original_q_len):
        self.got = layer_idx, tuple(k_exact.shape), original_q_len


def test_other_caches_get_what_they_got():
    from deltaattention_amd import attention
    cache, k, q = _OtherCache(), torch.zeros(1, 2, 10, 32), torch.zeros(1, 4, 10, 32)
    attention._handoff(cache, 1, _packed(), k, k, q, 0.1)
    assert cache.got == (1, (1, 2, 4, 32), 10)


@pytest.mark.parametrize("budget", [None, 4])
def test_four_bit_cache_gets_mass_with_a_budget(monkeypatch, budget):
    from deltaattention_amd import attention, ops
    from deltaattention_amd.deltaDecoding import FourBitCompressedCache
    cache = FourBitCompressedCache.__new__(FourBitCompressedCache)
    cache.budget, cache.observe, cache.exact_window_size = budget, 3, 4
    got = {}
    monkeypatch.setattr(FourBitCompressedCache, "initialize_from_prefill", lambda self, **kw: got.update(kw))
    monkeypatch.setattr(ops, "attention_mass", lambda q, k, **kw: ("mass", q.shape[2], kw["q_start"], kw["scale"]))
    k, q = torch.zeros(1, 2, 10, 32), torch.zeros(1, 4, 10, 32)
    attention._handoff(cache, 0, _packed(), k, k, q, 0.1)
    assert got.get("mass") == (None if budget is None else ("mass", 3, 7, 0.1))


def test_swap_hands_queries_to_the_bounded_cache_alone(monkeypatch):
    """PATH 2's hand-off of a full-width cache that carries a ``budget`` of its own."""
    from test_swap_flow import _stub, _tiny_model
    from deltaattention_amd import globVR
    from deltaattention_amd.deltaDecoding import HybridCompressedCache

    class Own(HybridCompressedCache):
        budget = 7

    monkeypatch.setattr(globVR, "delta_decode", True, raising=False)
    monkeypatch.setattr(globVR, "time_internal", False, raising=False)
    cfg, model = _tiny_model("deltaattention_dense")
    calls = _stub(monkeypatch)
    cache = Own(cfg, 1, dtype=torch.float32, exact_window_size=4, initial_capacity=16, device="cpu")
    with torch.no_grad():
        model.model(input_ids=torch.randint(0, 64, (1, 10)), past_key_values=cache, use_cache=True)
    assert [c[0] for c in calls] == ["dense", "handoff", "dense", "handoff"]
