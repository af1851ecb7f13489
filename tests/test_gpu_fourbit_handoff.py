"""FourBitCompressedCache.initialize_from_prefill: what a refused hand-off leaves behind."""
import pytest
import torch

from conftest import announce
from test_gpu_fourbit_steps import D, H, W, _cache, _state, _token, knobs  # noqa: F401 (knobs: autouse)

pytestmark = pytest.mark.gpu


def _args(gpu, gen, N=40):
    rows = [torch.randn(1, H, N, D, generator=gen).bfloat16().to(gpu) for _ in range(2)]
    ones = torch.ones(1, H, N, dtype=torch.int32, device=gpu)
    return dict(k_packed=rows[0], v_packed=rows[1], counts=ones, timestamps=ones.cumsum(-1).int(), k_exact=rows[0][:, :, -W:],
                v_exact=rows[1][:, :, -W:], original_q_len=N, mass=torch.rand(1, H, N, generator=gen).to(gpu))


@pytest.mark.parametrize("kind", ["no mass", "mass shape", "value rows", "sequences", "heads", "head dim", "type", "ring rows",
                                  "ring and values", "counts shape", "timestamps shape"])
def test_a_refused_handoff_changes_nothing(gpu, kind):
    announce(f"refused hand-off: {kind}")
    how = dict(budget=20, sinks=2, recent=4, slack=3, fill=3)
    cache, gen = _cache(gpu, **how)
    twin, _ = _cache(gpu, **how)
    before = _state(cache)
    good = _args(gpu, gen)
    bad = dict(good)
    if kind == "no mass":
        bad["mass"] = None
    elif kind == "mass shape":
        bad["mass"] = good["mass"][:, :, :-1].contiguous()
    elif kind == "value rows":
        bad["v_packed"] = good["v_packed"][:, :, :-1]
    elif kind == "type":
        bad["k_packed"], bad["v_packed"] = good["k_packed"].double(), good["v_packed"].double()
    elif kind == "ring rows":
        bad["k_exact"] = bad["v_exact"] = good["k_packed"][:, :, :W + 1]
    elif kind == "ring and values":
        bad["v_exact"] = good["v_exact"][:, :, :W - 1]
    elif kind in ("counts shape", "timestamps shape"):
        name = kind.split()[0]
        bad[name] = torch.cat([good[name]] * 2, 0)
    else:
        dim = {"sequences": 0, "heads": 1, "head dim": 3}[kind]
        for n in ("k_packed", "v_packed", "k_exact", "v_exact"):
            bad[n] = torch.cat([good[n]] * 2, dim)
        if dim < 2:
            for n in ("counts", "timestamps", "mass"):
                bad[n] = torch.cat([good[n]] * 2, dim)
    with pytest.raises((ValueError, TypeError)):
        cache.initialize_from_prefill(0, **bad)
    for x, y in zip(before, _state(cache)):
        assert torch.equal(x, y)
    # the cache goes on as if nothing had been asked, and takes a good prompt
    token = _token(gpu, gen)
    assert torch.equal(cache.decode_step(*token, 0), twin.decode_step(*token, 0))
    for c in (cache, twin):
        c.initialize_from_prefill(0, **good)
    assert torch.equal(cache.decode_step(*token, 0), twin.decode_step(*token, 0))
    for x, y in zip(_state(cache), _state(twin)):
        assert torch.equal(x, y)
