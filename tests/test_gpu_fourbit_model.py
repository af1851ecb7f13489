"""A model that decodes over FourBitCompressedCache through the swap: every layer's attention against 64
bits over what its cache holds, its way into the output projection, and layer 0's state against a
full-width cache fed by the same model."""
import pytest
import torch

from conftest import announce
from test_gpu_fourbit_cache import _attention, knobs  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

N, STEPS, W = 300, 40, 24


@pytest.mark.parametrize("impl,budget", [("deltaattention", None), ("deltaattention", 40), ("deltaattention_dense", None),
                                         ("deltaattention_dense", 40)])
def test_model_attention(gpu, knobs, impl, budget):  # noqa: F811
    import test_gpu_swap as S
    from deltaattention_amd.deltaDecoding import FourBitCompressedCache, HybridCompressedCache
    knobs.delta_decode, knobs.row_delta_threshold, knobs.row_similarity_metric = True, 8.0, "euclidean"
    knobs.packing_mode, knobs.target_keep_rate, knobs.time_internal = "periodic", 0.25, False
    seen = []

    class Checked(FourBitCompressedCache):
        def decode_step(self, q, k, v, layer_idx, scaling=None):
            assert scaling == pytest.approx(self.head_dim ** -0.5)
            out = super().decode_step(q, k, v, layer_idx, scaling=scaling)
            slot = (self.exact_seq_lens[layer_idx] - 1) % W
            assert torch.equal(self.k_exact[layer_idx, :, :, slot], k[:, :, 0])
            assert torch.equal(self.v_exact[layer_idx, :, :, slot], v[:, :, 0])
            want, tol, _, _ = _attention(q, self, layer_idx)
            assert ((out[:, :, 0].cpu().double() - want).abs() <= tol).all()
            seen.append(out)
            return out

    model = S._tiny_llama(impl)
    into = []
    hooks = [m.self_attn.o_proj.register_forward_pre_hook(lambda _, args: into.append(args[0])) for m in model.model.layers]
    ids = torch.randint(0, 512, (2, N + STEPS), generator=torch.Generator().manual_seed(6)).cuda()
    announce(f"four-bit model attention {impl} budget={budget}")
    more = {} if budget is None else dict(budget=budget, sinks=2, recent=8, slack=6)
    cache = Checked(model.config, 2, dtype=torch.bfloat16, exact_window_size=W, **more)
    full = HybridCompressedCache(model.config, 2, dtype=torch.bfloat16, exact_window_size=W)
    with torch.no_grad():
        for c in (cache, full):
            first = model(ids[:, :N], past_key_values=c, use_cache=True).logits
            if c is cache:
                logits = first
        assert torch.equal(first, logits)  # the prompt's pass does not depend on the cache
        for t in range(N, N + STEPS):
            at = dict(use_cache=True, position_ids=torch.tensor([[t]], device=gpu))
            seen.clear(), into.clear()
            model(ids[:, t:t + 1], past_key_values=cache, **at)
            assert len(seen) == len(into) == 2
            for out, got in zip(seen, into):
                assert torch.equal(out.transpose(1, 2).reshape(2, 1, -1), got)
            model(ids[:, t:t + 1], past_key_values=full, **at)
    for h in hooks:
        h.remove()
    # layer 0's keys and values do not depend on any attention
    assert torch.equal(cache.k_exact[0], full.k_exact[0]) and torch.equal(cache.v_exact[0], full.v_exact[0])
    assert cache.total_seq_lens == full.total_seq_lens == [N + STEPS] * 2
    if impl == "deltaattention" and budget is None:  # every head the same anchors: no padding in the full cache
        kv = cache.anchors[0]
        for b in range(2):
            for h in range(2):
                n = int(kv.lengths[b, h])
                assert n == int(full.packed_lengths[0, 2 * b + h])
                assert torch.equal(kv.counts[b, h, :n], full.packed_counts[0, b, h, :n])
                assert torch.equal(kv.timestamps[b, h, :n], full.packed_timestamps[0, b, h, :n])
    if budget is not None:
        for kv in cache.anchors:
            assert int(kv.lengths.max()) <= budget + 6 and float(kv.mass.sum()) > 0
