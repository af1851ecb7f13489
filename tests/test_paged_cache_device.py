"""A PagedCache stays on the device that was current when it was made."""
import types

import pytest
import torch

from conftest import announce


def test_device_of_a_cache(monkeypatch):
    """Its later tensors are made there whatever device is current then: the device has its index."""
    from deltaattention_amd import paged_cache
    made = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(paged_cache, "_Pool", lambda *a: made.append(a[-1]) or types.SimpleNamespace(raw=0, drop=len))
    monkeypatch.setattr(torch, "zeros", lambda *a, device=None, **k: made.append(device))
    config = types.SimpleNamespace(head_dim=64, num_key_value_heads=2, num_hidden_layers=1, hidden_size=256,
                                   num_attention_heads=4)
    for given, want in (("cuda", 3), ("cuda:1", 1), (torch.device("cuda"), 3)):
        made.clear()
        cache = paged_cache.PagedCache(config, 2, device=given)
        assert cache.device == torch.device("cuda", want) and made == [torch.device("cuda", want)] * 3


@pytest.mark.gpu
def test_device_on_the_gpu(gpu):
    from deltaattention_amd.paged_cache import PagedCache
    announce("PagedCache: its device")
    config = types.SimpleNamespace(head_dim=64, num_key_value_heads=2, num_hidden_layers=1, hidden_size=256,
                                   num_attention_heads=4)
    cache = PagedCache(config, 2)
    x = torch.randn(2, 2, 300, 64, device="cuda").bfloat16()
    cache.append(x, x, 0)
    assert cache.device == cache._table.device == cache._pool.k.device == torch.device("cuda", torch.cuda.current_device())
    assert cache.fork(2).device == cache.device
