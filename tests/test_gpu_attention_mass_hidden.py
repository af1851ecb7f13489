"""Accumulated weights of keys that no query sees: they get 0 and disturb nothing, whatever they hold and
however the number of query rows lies to a stage of them."""
import math

import pytest
import torch

from conftest import announce
from test_gpu_attention_mass import DTYPES, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("stamped", [False, True])
@pytest.mark.parametrize("B,H,G,D,Nq,Nk", [(1, 1, 1, 64, 1, 40), (2, 2, 1, 128, 33, 300), (1, 2, 3, 72, 50, 700),
                                           (1, 1, 4, 128, 16, 300), (1, 2, 2, 64, 65, 2100), (1, 1, 7, 96, 100, 90)])
def test_keys_that_no_query_sees(gpu, B, H, G, D, Nq, Nk, stamped, dtype):
    from deltaattention_amd import ops
    gen = torch.Generator().manual_seed(Nq * 31 + Nk)
    dt = DTYPES[dtype]
    q = (1.5 * torch.randn(B, H * G, Nq, D, generator=gen)).to(dt)
    k = torch.randn(B, H, Nk, D, generator=gen).to(dt)
    start = 2 * Nk // 3 - Nq + 1  # without timestamps the last third lies behind every query
    when = torch.arange(Nk).expand(B, H, Nk)
    ts = None
    if stamped:  # hidden keys anywhere among the others, one at the latest time there is
        late = torch.rand(B, H, Nk, generator=gen) < 0.3
        late[..., 0] = False
        when = torch.where(late, start + Nq + torch.randint(0, 50, (B, H, Nk), generator=gen), when.clamp(max=max(start, 0)))
        when[..., -1] = 2 ** 31 - 1
        ts = when.int().contiguous()
    hidden = when > start + Nq - 1
    assert hidden.any() and not hidden.all()
    want, bound = _want(q, torch.where(hidden[..., None], torch.zeros((), dtype=dt), k), None, ts, None, start)
    k = k.clone()
    k[hidden] = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dt).min] * (D // 4)).to(dt)
    announce(f"mass hidden keys {dtype} {Nq}x{Nk} stamped={stamped}")
    got = ops.attention_mass(q.to(gpu), k.to(gpu), timestamps=None if ts is None else ts.to(gpu), q_start=start).cpu().double()
    assert (got[hidden] == 0).all(), got[hidden]
    off = (got - want).abs()
    assert (off <= bound).all(), f"{(off / bound).max():.3g} of the bound"
