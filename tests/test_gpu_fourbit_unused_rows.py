"""Rows of a FourBitCompressedCache that no anchor has taken yet have no accumulated weight, whatever
their memory held before."""
import types

import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("budget", [None, 24])
def test_unused_rows_have_no_mass(gpu, budget):
    from deltaattention_amd import globVR
    from deltaattention_amd.deltaDecoding import FourBitCompressedCache
    announce(f"four-bit cache: mass of unused rows, budget={budget}")
    junk = [torch.full((1 << 16,), float("nan"), device=gpu) for _ in range(8)]  # what the allocator gives out next
    del junk
    cfg = types.SimpleNamespace(head_dim=64, num_key_value_heads=2, num_hidden_layers=1, hidden_size=256,
                                num_attention_heads=4)
    more = {} if budget is None else dict(budget=budget, sinks=2, recent=4, slack=8)
    cache = FourBitCompressedCache(cfg, 1, dtype=torch.bfloat16, exact_window_size=8, initial_capacity=64, **more)
    gen = torch.Generator().manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16).cuda()  # noqa: E731
    assert (cache.anchors[0].mass == 0).all()
    P = 40
    counts = torch.ones(1, 2, P, dtype=torch.int32, device=gpu)
    stamps = torch.arange(P, dtype=torch.int32, device=gpu).expand(1, 2, P).contiguous()
    mass = torch.rand(1, 2, P, generator=gen).cuda()
    cache.initialize_from_prefill(0, rand(1, 2, P, 64), rand(1, 2, P, 64), counts, stamps, rand(1, 2, 8, 64),
                                  rand(1, 2, 8, 64), P, mass=mass)
    saved = globVR.row_delta_threshold, globVR.row_similarity_metric
    globVR.row_delta_threshold, globVR.row_similarity_metric = 0.0, "euclidean"  # every evicted token a new anchor
    try:
        for _ in range(25):
            kv = cache.anchors[0]
            n = int(kv.lengths.max())
            assert torch.isfinite(kv.mass).all() and (kv.mass[:, :, n:] == 0).all() and (kv.mass[:, :, :n] >= 0).all()
            cache.decode_step(rand(1, 4, 1, 64), rand(1, 2, 1, 64), rand(1, 2, 1, 64), 0)
    finally:
        globVR.row_delta_threshold, globVR.row_similarity_metric = saved
