"""FourBitCompressedCache's decode steps: what a refused call leaves behind."""
from types import SimpleNamespace

import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu

Hq, H, D, W = 8, 2, 64, 8


def _cache(gpu, budget=None, tokens=40, fill=0, **more):
    """A cache after a prompt of ``tokens`` tokens that are all anchors, and ``fill`` decode tokens."""
    from deltaattention_amd import globVR
    from deltaattention_amd.deltaDecoding import FourBitCompressedCache
    cfg = SimpleNamespace(hidden_size=Hq * D, num_attention_heads=Hq, num_key_value_heads=H, num_hidden_layers=1, head_dim=D)
    cache = FourBitCompressedCache(cfg, 1, dtype=torch.bfloat16, exact_window_size=W, budget=budget, **more)
    gen = torch.Generator().manual_seed(tokens)
    rows = [torch.randn(1, H, tokens, D, generator=gen).bfloat16().to(gpu) for _ in range(2)]
    ones = torch.ones(1, H, tokens, dtype=torch.int32, device=gpu)
    at = torch.arange(tokens, dtype=torch.int32, device=gpu).expand(1, H, tokens)
    cache.initialize_from_prefill(0, *rows, ones, at, *(x[:, :, -W:] for x in rows), tokens,
                                  **({} if budget is None else {"mass": torch.rand(1, H, tokens, generator=gen).to(gpu)}))
    globVR.row_delta_threshold, globVR.row_similarity_metric = 0.0, "euclidean"  # every token is an anchor
    for _ in range(fill):
        cache.decode_step(*_token(gpu, gen), 0)
    return cache, gen


@pytest.fixture(autouse=True)
def knobs():
    from deltaattention_amd import globVR
    saved = dict(vars(globVR))
    yield
    for name, val in saved.items():
        setattr(globVR, name, val)


def _token(gpu, gen):
    return [torch.randn(1, h, 1, D, generator=gen).bfloat16().to(gpu) for h in (Hq, H, H)]


def _state(cache):
    kv = cache.anchors[0]
    n = int(kv.lengths.max())
    held = [getattr(kv, name)[:, :, :n].clone() for name in ("k_codes", "k_scales", "v_codes", "v_scales", "counts",
                                                             "timestamps", "mass")]
    return held + [kv.lengths.clone(), cache.k_last.clone(), cache.k_exact.clone(), cache.v_exact.clone(),
                   torch.tensor([cache.exact_seq_lens[0], cache.total_seq_lens[0], cache.max_packed_len[0], kv.capacity])]


def _bad(kind, q, k, v):
    """(query, key, value, scaling) of a call that has to be refused."""
    scaling = None
    if kind == "query type":
        q = q.float()
    elif kind == "query heads":
        q = torch.cat([q, q], 1)[:, :Hq + 1]
    elif kind == "query group":
        q = q.expand(1, Hq, 1, D).repeat(1, 65 * H // Hq + 1, 1, 1)[:, :65 * H]
    elif kind == "query tokens":
        q = torch.cat([q, q], 2)
    elif kind == "query dims":
        q = q[..., :D - 8]
    elif kind == "query batch":
        q = torch.cat([q, q], 0)
    elif kind == "query device":
        q = q.cpu()
    elif kind == "scaling":
        scaling = 0.0
    elif kind == "scaling nan":
        scaling = float("nan")
    elif kind == "key type":
        k, v = k.float(), v.float()
    elif kind == "key tokens":
        k, v = torch.cat([k, k], 2), torch.cat([v, v], 2)
    elif kind == "value dims":
        v = v[..., :D - 8]
    return q, k, v, scaling


KINDS = ["query type", "query heads", "query group", "query tokens", "query dims", "query batch", "query device", "scaling",
         "scaling nan", "key type", "key tokens", "value dims"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", ["plain", "full", "cut due"])
def test_a_refused_step_changes_nothing(gpu, kind, form):
    """``full``: no row is free, the next token grows the cache; ``cut due``: it cuts to the budget.  The
    step that follows the refusal gives what it gives without one."""
    announce(f"refused step: {kind}, {form}")
    how = {"plain": dict(fill=3), "full": dict(initial_capacity=1, tokens=40, fill=1024),
           "cut due": dict(budget=20, sinks=2, recent=4, slack=3, fill=3)}[form]
    cache, gen = _cache(gpu, **how)
    twin, _ = _cache(gpu, **how)
    if form != "plain":
        assert cache.max_packed_len[0] == cache.anchors[0].capacity
    before = _state(cache)
    q, k, v = _token(gpu, gen)
    bad_q, bad_k, bad_v, scaling = _bad(kind, q, k, v)
    with pytest.raises((ValueError, TypeError)):
        cache.decode_step(bad_q, bad_k, bad_v, 0, scaling)
    for x, y in zip(before, _state(cache)):
        assert torch.equal(x, y)
    assert torch.equal(cache.decode_step(q, k, v, 0), twin.decode_step(q, k, v, 0))
    for x, y in zip(_state(cache), _state(twin)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("kind", ["key type", "value dims"])
def test_a_refused_update_changes_nothing(gpu, kind):
    """``update`` alone, with a cut due."""
    announce(f"refused update: {kind}")
    cache, gen = _cache(gpu, budget=20, sinks=2, recent=4, slack=3, fill=3)
    before, held = _state(cache), cache.anchors[0]
    q, k, v = _token(gpu, gen)
    _, bad_k, bad_v, _ = _bad(kind, q, k, v)
    with pytest.raises((ValueError, TypeError)):
        cache.update(bad_k, bad_v, 0)
    assert cache.anchors[0] is held
    for x, y in zip(before, _state(cache)):
        assert torch.equal(x, y)
