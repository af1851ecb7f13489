"""Decode attention over 4-bit rows and accumulated weights use every bf16 part that they name
(kv4_precision: limits that a kernel with a part less exceeds)."""
import pytest
import torch

import kv4_precision as P
import kv4_reference as ref
from conftest import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,H,G,D,n", [(1, 2, 4, 128, 600), (1, 1, 8, 64, 5000), (2, 2, 1, 96, 97), (1, 1, 20, 128, 700)])
def test_attention_parts(gpu, B, H, G, D, n, dtype):
    from deltaattention_amd import ops
    q, k, v, counts = P.attention_inputs(B, H, G, D, n, dtype, n + D)
    kc, ks = ref.encode(k)
    vc, vs = ref.encode(v)
    k, v = ref.decode(kc, ks, D).float(), ref.decode(vc, vs, D).float()
    lengths = torch.full((B, H), n, dtype=torch.int32)
    dev = [x.to(gpu) for x in (kc, ks, vc, vs, counts, torch.zeros_like(counts), lengths)]
    kv = ops.KV4(*dev, D, torch.zeros(B, H, n, device=gpu))
    announce(f"attention parts {dtype} n={n}")
    for accumulate in (False, True):  # with weights a form of its own
        out = ops.decode_attention_kv4(q.to(gpu), kv, accumulate=accumulate).cpu()
        P.assert_attention(out, kv.mass.cpu() if accumulate else None, q, k, v, counts, dtype)


@pytest.mark.parametrize("B,H,G,D,Nq,Nk", [(1, 2, 1, 128, 1, 600), (1, 1, 4, 64, 7, 300), (2, 1, 2, 96, 40, 90),
                                           (1, 2, 4, 128, 64, 5000)])
def test_mass_parts(gpu, B, H, G, D, Nq, Nk):
    from deltaattention_amd import ops
    q, k = P.mass_inputs(B, H, G, D, Nq, Nk, seed=Nk)
    announce(f"mass parts {Nq}x{Nk}")
    got = ops.attention_mass(q.to(gpu), k.to(gpu), q_start=Nk).cpu()
    P.assert_mass(got, q, k)
