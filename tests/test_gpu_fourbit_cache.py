"""FourBitCompressedCache: prefill hand-off, decode steps and cuts to the budget, against the oracle's
state machine (decisions at full width), the 4-bit format and attention in 64 bits."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import kv4_reference as ref
import test_gpu_dropin as T
from conftest import announce, oracle_arith
from oracle import delta_oracle as O
from oracle import select_oracle_c as OC

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture
def knobs():
    from deltaattention_amd import globVR
    saved = dict(vars(globVR))
    globVR.packing_mode, globVR.chunk_size, globVR.time_internal = "delta", 512, False
    yield globVR
    for name, val in saved.items():
        setattr(globVR, name, val)


def _config(Hq, Hkv, D, layers=1):
    return SimpleNamespace(hidden_size=Hq * D, num_attention_heads=Hq, num_key_value_heads=Hkv,
                           num_hidden_layers=layers, head_dim=D)


def _inputs(B, Hq, Hkv, N, D, dtype, seed):
    from deltaattention_amd import synth
    return (t.to(DTYPES[dtype]) for t in synth.make_layer_inputs(B, Hq, Hkv, N, D, seed=seed, rope_base=10000.0))


def _attention(q, cache, layer=0):
    """The layer's attention in 64 bits over what its cache holds, with its bound (see ref.attention)."""
    kv = cache.anchors[layer]
    B, H, D = kv.batch, kv.kv_heads, kv.head_dim
    G = q.shape[1] // H
    W = min(cache.exact_seq_lens[layer], cache.exact_window_size)
    kf, vf = ref.decode(kv.k_codes, kv.k_scales, D), ref.decode(kv.v_codes, kv.v_scales, D)
    want, tol, weights, wtol = (torch.zeros(s).double() for s in ((B, H * G, D), (B, H * G, D), (B, H, kv.capacity),
                                                                  (B, H, kv.capacity)))
    eps = torch.finfo(q.dtype).eps / 2
    for b in range(B):
        for h in range(H):
            n = int(kv.lengths[b, h])
            k = torch.cat([kf[b, h, :n], cache.k_exact[layer, b, h, :W].cpu().double()])
            v = torch.cat([vf[b, h, :n], cache.v_exact[layer, b, h, :W].cpu().double()])
            size = torch.cat([kv.counts[b, h, :n].cpu().clamp(min=0).double(), torch.ones(W).double()])
            sl = slice(h * G, (h + 1) * G)
            o, w, spread, drift = ref.attention(q[b, sl, 0].cpu().double(), k, v, size)
            rel = drift[:, None] + 2.0 ** -16 * (q.dtype != torch.float32) + (n + W + 64) * 2.0 ** -24
            want[b, sl], tol[b, sl] = o, eps * o.abs() + (1 + eps) * rel * spread + 1e-30
            weights[b, h, :n] = w[:, :n].sum(0)
            wtol[b, h, :n] = (w[:, :n] * (drift[:, None] + (n + W + 64) * 2.0 ** -24)).sum(0)
    return want, tol, weights, wtol


@pytest.mark.parametrize("B,Hkv,G,D,N,W,steps,metric,tau,dtype,cap0", [
    (1, 2, 4, 128, 700, 50, 70, "euclidean", 10.0, "bf16", 64), (2, 3, 2, 64, 500, 16, 60, "cosine", 0.85, "fp16", 16),
    (1, 2, 1, 96, 600, 128, 40, "euclidean", 9.0, "fp32", 1024), (1, 1, 8, 40, 300, 20, 90, "euclidean", 3.0, "bf16", 300),
    (1, 2, 4, 128, 20, 64, 60, "cosine", 0.99, "bf16", 8)])
def test_decode_decisions(gpu, knobs, B, Hkv, G, D, N, W, steps, metric, tau, dtype, cap0):
    """Unbounded: counts, timestamps, lengths and ring bit for bit the full-width state machine's
    (each head with its own anchors), rows its rows in 4 bits, attention within its bound."""
    from deltaattention_amd import attention
    from deltaattention_amd.deltaDecoding import FourBitCompressedCache
    knobs.row_delta_threshold, knobs.row_similarity_metric = tau, metric
    q, k, v = _inputs(B, Hkv * G, Hkv, N + steps, D, dtype, N + D)
    announce(f"four-bit decode {metric} {dtype} D={D} N={N}")
    cache = FourBitCompressedCache(_config(Hkv * G, Hkv, D), B, dtype=DTYPES[dtype], exact_window_size=W,
                                   initial_capacity=cap0)
    qg, kg, vg = q.to(gpu), k.to(gpu), v.to(gpu)
    attention.delta_prefill_attention(qg[:, :, :N], kg[:, :, :N], vg[:, :, :N], 0, cache)
    kf, vf = k.float().numpy(), v.float().numpy()
    keep, _ = OC.select_delta(kf[:, :, :N], tau, 512, 0, metric, arith=oracle_arith(k))
    p = O.pack(kf[:, :, :N], vf[:, :, :N], keep)
    st = T._oracle_cache_from_prefill(p, kf[:, :, :N], vf[:, :, :N], W, N + steps + 1)
    st["lengths"][:] = (p["counts"] > 0).sum(-1).reshape(-1)
    for t in range(steps):
        sl = slice(N + t, N + t + 1)
        out = cache.decode_step(qg[:, :, sl], kg[:, :, sl], vg[:, :, sl], 0)
        O.decode_update(st, kf[:, :, sl], vf[:, :, sl], tau, metric)
        if t % 23 == 0 or t == steps - 1:
            want, tol, _, _ = _attention(q[:, :, sl], cache)
            assert ((out[:, :, 0].cpu().double() - want).abs() <= tol).all(), t
    kv = cache.anchors[0]
    assert (cache.packed_lengths[0].cpu().numpy() == st["lengths"]).all()
    assert torch.equal(cache.k_exact[0].float().cpu(), torch.from_numpy(st["k_exact"]))
    assert torch.equal(cache.v_exact[0].float().cpu(), torch.from_numpy(st["v_exact"]))
    assert cache.get_seq_length(0) == N + steps
    for b in range(B):
        for h in range(Hkv):
            n = int(st["lengths"][b * Hkv + h])
            assert (kv.counts[b, h, :n].cpu().numpy() == st["counts"][b, h, :n]).all()
            assert (kv.timestamps[b, h, :n].cpu().numpy() == st["timestamps"][b, h, :n]).all()
            for codes, scales, rows in ((kv.k_codes, kv.k_scales, st["k_packed"]), (kv.v_codes, kv.v_scales, st["v_packed"])):
                want_c, want_s = ref.encode(torch.from_numpy(rows[b, h, :n]))
                assert torch.equal(codes[b, h, :n].cpu(), want_c) and torch.equal(scales[b, h, :n].cpu(), want_s)
            assert torch.equal(cache.k_last[0, b, h].float().cpu(), torch.from_numpy(st["k_packed"][b, h, n - 1]))


@pytest.mark.parametrize("B,Hkv,G,D,N,dtype,budget,sinks,recent,slack,observe", [
    (1, 2, 4, 128, 600, "bf16", 48, 4, 16, 7, 64), (2, 2, 2, 64, 300, "fp32", 20, 0, 1, 1, 1000),
    (1, 1, 3, 80, 40, "fp16", 64, 2, 8, 5, 16)])
def test_bounded(gpu, knobs, B, Hkv, G, D, N, dtype, budget, sinks, recent, slack, observe):
    """Prompt weights, the cut at the hand-off, weights added by every token, cuts while decoding: each
    step's state follows from the one before it by the plain rules."""
    from deltaattention_amd import attention, ops
    from deltaattention_amd.deltaDecoding import FourBitCompressedCache, decode_attention
    knobs.row_delta_threshold, knobs.row_similarity_metric = 6.0 * (D / 128) ** 0.5, "euclidean"
    W, steps = 24, 60
    q, k, v = _inputs(B, Hkv * G, Hkv, N + steps, D, dtype, budget)
    qg, kg, vg = q.to(gpu), k.to(gpu), v.to(gpu)
    announce(f"four-bit bounded {dtype} D={D} budget={budget}")
    cache = FourBitCompressedCache(_config(Hkv * G, Hkv, D), B, dtype=DTYPES[dtype], exact_window_size=W, budget=budget,
                                   sinks=sinks, recent=recent, slack=slack, observe=observe)
    attention.delta_prefill_attention(qg[:, :, :N], kg[:, :, :N], vg[:, :, :N], 0, cache)
    # the hand-off, from its own parts
    keep, _ = ops.select(kg[:, :, :N], knobs.row_delta_threshold, 512)
    pk = ops.pack(keep, kg[:, :, :N], vg[:, :, :N]).trimmed()
    n_obs = min(observe, N)
    mass = ops.attention_mass(qg[:, :, N - n_obs:N], pk.k_packed, pk.counts.contiguous(), pk.timestamps.contiguous(),
                              pk.anchor_counts, q_start=N - n_obs).cpu()
    kv = cache.anchors[0]
    for b in range(B):
        for h in range(Hkv):
            rows = ref.heavy(mass[b, h].tolist(), int(pk.anchor_counts[b, h]), budget, sinks, recent)
            assert int(kv.lengths[b, h]) == len(rows)
            assert torch.equal(kv.timestamps[b, h, :len(rows)].cpu(), pk.timestamps[b, h].cpu()[rows])
            assert torch.equal(kv.mass[b, h, :len(rows)].cpu(), mass[b, h][rows])
            want_c, _ = ref.encode(pk.k_packed[b, h].cpu()[rows])
            assert torch.equal(kv.k_codes[b, h, :len(rows)].cpu(), want_c)
    cuts = 0
    for t in range(steps):
        sl = slice(N + t, N + t + 1)
        old = cache.anchors[0]
        before = {n: getattr(old, n).cpu().clone() for n in ("counts", "timestamps", "mass", "k_codes")}
        lens = old.lengths.cpu().clone()
        cache.update(kg[:, :, sl], vg[:, :, sl], 0)
        new = cache.anchors[0]
        cut = new is not old
        cuts += cut
        for b in range(B):
            for h in range(Hkv):
                n = int(lens[b, h])
                rows = ref.heavy(before["mass"][b, h].tolist(), n, budget, sinks, recent) if cut else list(range(n))
                m = int(new.lengths[b, h])
                assert len(rows) <= m <= len(rows) + 1 <= budget + slack
                for name in ("timestamps", "mass", "k_codes"):
                    assert torch.equal(getattr(new, name)[b, h, :len(rows)].cpu(), before[name][b, h][rows]), (t, name)
                grown = int(new.counts[b, h, :len(rows)].sum()) - int(before["counts"][b, h][rows].sum())
                assert grown + (m - len(rows)) == (1 if cache.exact_seq_lens[0] > W else 0)
                if m > len(rows):
                    assert int(new.counts[b, h, m - 1]) == 1 and float(new.mass[b, h, m - 1]) == 0.0
                    assert int(new.timestamps[b, h, m - 1]) == N + t - W
        start = new.mass.cpu().double()
        out = decode_attention(qg[:, :, sl], cache, 0)
        if t % 9 == 0 or cut:
            want, tol, weights, wtol = _attention(q[:, :, sl], cache)
            assert ((out[:, :, 0].cpu().double() - want).abs() <= tol).all(), t
            live = torch.arange(new.capacity) < new.lengths.cpu()[..., None]
            off = (new.mass.cpu().double() - start - weights).abs()
            assert (off <= wtol + 2.0 ** -23 * (start + weights))[live].all(), t
    # every token past the ring's window may add a row, so the room is made in time
    evictions = max(0, min(N, W) + steps - W)
    if min(pk.k_packed.shape[2], budget) + evictions > budget + slack + 1:
        assert cuts > 0


def test_handoff_refusals(gpu):
    from deltaattention_amd.deltaDecoding import FourBitCompressedCache
    cfg = _config(4, 2, 64)
    for bad in (dict(budget=10, sinks=8, recent=4), dict(budget=10, recent=0), dict(budget=100, slack=0),
                dict(budget=100, observe=0)):
        with pytest.raises(ValueError):
            FourBitCompressedCache(cfg, 1, **bad)
    cache = FourBitCompressedCache(cfg, 1, dtype=torch.bfloat16, exact_window_size=8, budget=4, sinks=1, recent=1)
    rows = torch.randn(1, 2, 9, 64, device=gpu).bfloat16()
    ones = torch.ones(1, 2, 9, dtype=torch.int32, device=gpu)
    with pytest.raises(ValueError, match="mass"):
        cache.initialize_from_prefill(0, rows, rows, ones, ones, rows[:, :, :8], rows[:, :, :8], 9)


@pytest.mark.parametrize("impl", ["deltaattention", "deltaattention_dense"])
def test_model(gpu, knobs, impl):
    """A small Llama prefills and decodes over a bounded 4-bit cache through the swap: the anchors stay
    within the budget, gather weight, and the logits are finite."""
    import test_gpu_swap as S
    from deltaattention_amd.deltaDecoding import FourBitCompressedCache
    knobs.delta_decode, knobs.row_delta_threshold, knobs.row_similarity_metric = True, 8.0, "euclidean"
    model = S._tiny_llama(impl)
    ids = torch.randint(0, 512, (1, 400), generator=torch.Generator().manual_seed(5)).cuda()
    announce(f"four-bit model {impl}")
    cache = FourBitCompressedCache(model.config, 1, dtype=torch.bfloat16, exact_window_size=32, budget=96, recent=16, slack=8)
    with torch.no_grad():
        model(ids, past_key_values=cache, use_cache=True)
        for t in range(24):
            knobs.time_internal = t % 5 == 4  # the stage-timed way runs update and attention apart
            out = model(ids[:, t:t + 1], past_key_values=cache, use_cache=True,
                        position_ids=torch.tensor([[400 + t]], device=gpu))
            assert torch.isfinite(out.logits).all(), t
    assert cache.get_seq_length(0) == 424
    for layer in range(2):
        assert 0 < int(cache.packed_lengths[layer].max()) <= 104
        assert float(cache.anchors[layer].mass[:, :, :16].sum()) > 0


def test_deepcopy(gpu, knobs):
    """A prompt's cache can be copied and continued twice: the copies share nothing."""
    import copy
    from deltaattention_amd import attention
    from deltaattention_amd.deltaDecoding import FourBitCompressedCache
    knobs.row_delta_threshold, knobs.row_similarity_metric = 6.0, "euclidean"
    Hkv, G, D, N, W = 2, 4, 64, 300, 16
    q, k, v = (t.to(gpu) for t in _inputs(1, Hkv * G, Hkv, N + 30, D, "bf16", 3))
    announce("four-bit deepcopy")
    cache = FourBitCompressedCache(_config(Hkv * G, Hkv, D), 1, dtype=torch.bfloat16, exact_window_size=W, budget=64,
                                   recent=16, slack=8)
    attention.delta_prefill_attention(q[:, :, :N], k[:, :, :N], v[:, :, :N], 0, cache)
    bare = cache.anchors[0]
    twin = copy.deepcopy(cache)
    outs = []
    for c in (cache, twin):
        before = bare.lengths.clone(), bare.mass.clone()
        outs.append([c.decode_step(q[:, :, t:t + 1], k[:, :, t:t + 1], v[:, :, t:t + 1], 0) for t in range(N, N + 30)])
        if c is twin:
            assert torch.equal(bare.lengths, before[0]) and torch.equal(bare.mass, before[1])
    for x, y in zip(*outs):
        assert torch.equal(x, y)
    assert copy.deepcopy(bare).mass.data_ptr() != bare.mass.data_ptr()
