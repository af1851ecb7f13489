"""copy.copy, pickle and torch.save of a KV4, and of the cache that holds some."""
import copy
import io
import pickle

import pytest
import torch

from conftest import announce
from test_gpu_fourbit_steps import _cache, _token, knobs  # noqa: F401 (knobs: autouse)

pytestmark = pytest.mark.gpu

NAMES = ("k_codes", "k_scales", "v_codes", "v_scales", "counts", "timestamps", "lengths")


@pytest.mark.parametrize("mass", [True, False])
@pytest.mark.parametrize("made", ["empty", "tensors"])
def test_copies_of_a_cache(gpu, made, mass):
    from deltaattention_amd import ops
    announce(f"KV4 copies {made} mass={mass}")
    gen = torch.Generator().manual_seed(8)
    rows = torch.randn(2, 3, 20, 40, generator=gen).to(gpu)
    made_kv = ops.quantize_kv4(rows, rows, capacity=24)
    names = NAMES + ("mass",) * mass
    if made == "empty":
        kv = ops.KV4.empty(2, 3, 24, 40, gpu, mass=mass)
        for n in names:
            getattr(kv, n).copy_(getattr(made_kv, n))
    else:  # memory of their own, as a program that keeps its own tensors has them
        kv = ops.KV4(*(getattr(made_kv, n).clone() for n in NAMES), 40, made_kv.mass.clone() if mass else None)
    same = copy.copy(kv)
    assert same is not kv and type(same) is ops.KV4
    for n in names:
        assert getattr(same, n).data_ptr() == getattr(kv, n).data_ptr()
    again = pickle.loads(pickle.dumps(kv))
    held = io.BytesIO()
    torch.save(kv, held)
    held.seek(0)
    saved = torch.load(held, weights_only=False)  # this test's own bytes
    q = torch.randn(2, 6, 1, 40, generator=gen).to(gpu)
    want = ops.decode_attention_kv4(q, kv)
    for other in (same, again, saved):
        assert (other.batch, other.kv_heads, other.capacity, other.head_dim) == (2, 3, 24, 40)
        assert (other.mass is None) == (not mass)
        assert torch.equal(ops.decode_attention_kv4(q, other), want)
    for other in (again, saved):
        for n in names:
            a, b = getattr(other, n), getattr(kv, n)
            assert a.data_ptr() != b.data_ptr()
            if a.dim() > 2:  # rows past the lengths are undefined
                a, b = a[:, :, :20], b[:, :, :20]
            assert torch.equal(a, b)


def test_pickled_cache_continues(gpu):
    announce("four-bit cache pickled")
    cache, gen = _cache(gpu, budget=20, sinks=2, recent=4, slack=3, fill=3)
    twin = pickle.loads(pickle.dumps(cache))
    for _ in range(6):
        token = _token(gpu, gen)
        assert torch.equal(cache.decode_step(*token, 0), twin.decode_step(*token, 0))
