"""The model swap's step over a PagedCache (on the CPU, kernels replaced)."""
import types

import pytest
import torch

from paged_cache_on_cpu import cache, held, kernels, state, tokens  # noqa: F401 (kernels: a fixture)


def test_a_prompt_that_is_refused(kernels, monkeypatch):  # noqa: F811
    """PATH 1 refuses a prompt (a setting that it does not know, say): the cache is as before, and takes it later."""
    from deltaattention_amd import attention, llama_swap
    c = cache()
    layer = types.SimpleNamespace(config=types.SimpleNamespace(_attn_implementation=llama_swap.DELTA), layer_idx=0, scaling=0.25)
    q, (k, v) = tokens(2, 9, 4)[0], tokens(2, 9)
    cos, sin = torch.ones(1, 9, 16), torch.zeros(1, 9, 16)
    calls = []

    def prefill(query, key, value, out=None, **more):
        calls.append(more["layer_idx"])
        if len(calls) == 1:
            raise ValueError("packing_mode")
        out.copy_(query)
    monkeypatch.setattr(attention, "delta_prefill_attention", prefill)
    before = state(c)
    with pytest.raises(ValueError):
        llama_swap._paged_attention(layer, c, q, k, v, cos, sin)
    assert state(c) == before
    assert torch.equal(llama_swap._paged_attention(layer, c, q, k, v, cos, sin), q.transpose(1, 2))
    assert calls == [0, 0] and all(torch.equal(x, y) for x, y in zip(held(c), (k, v)))
