"""Paged attention where most of a result comes from weights that 16 bits hardly hold."""
import math

import pytest
import torch

import paged_reference as R
from conftest import announce

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _i(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("new,prefix", [(1, False), (40, False), (1, True), (40, True)])
def test_many_small_weights(gpu, new, prefix, dtype):
    """One key that a query likes best, with values of 0, and thousands of others at 2^-25.3 of its weight, whose
    values are the whole result."""
    from deltaattention_amd import ops
    announce(f"paged attention, small weights, {new} tokens, prefix={prefix} {dtype}")
    N, D, page = 4000, 64, 16
    P = N // page + new // page + 2
    k, v = (torch.zeros(P, 1, page, D, dtype=DT[dtype]) for _ in range(2))
    q = torch.zeros(4 * new, 2, D, dtype=DT[dtype])
    # score of the first key over the others': 25.3 in powers of two
    q[..., 0], k[..., 0] = 16.0, 0.0
    k[0, 0, 0, 0] = 8.0
    scale = 25.3 * math.log(2.0) / 128.0
    v[...] = 1.0 + torch.arange(D).to(DT[dtype]) / D
    v[0, 0, 0] = 0.0
    own = N + new if not prefix else new
    first = 0 if not prefix else N // page
    table = torch.arange(first, P, dtype=torch.int32)[None].repeat(4, 1).contiguous()
    kv = ops.PagedKV(k.cuda(), v.cuda())
    cu = [new * b for b in range(5)]
    batch = ops.PagedBatch(table.cuda(), _i([own] * 4), cu)
    pre = (torch.arange(N // page, dtype=torch.int32)[None], [N], [0, 4 * new]) if prefix else None
    if prefix:
        got = ops.shared_prefix_attention(q.cuda(), kv, batch, ops.PagedBatch(pre[0].cuda(), _i(pre[1]), pre[2]), scale=scale)
    else:
        got = ops.paged_attention(q.cuda(), kv, batch, scale=scale)
    want, tol = R.attention(q, k, v, table, [own] * 4, cu, pre, scale)
    assert want.abs().min() > 2.0 ** -14  # a normal number in every type, and not the best key's
    if dtype == "fp16":
        # a weight is held as 2^11 times its share of the largest at least: below 2^-14 of fp16's range it is off
        # by up to half of 2^-24, which is 2^-36 of the largest weight (at most 1) for each of the keys
        tol = tol + (N + new) * 2.0 ** -36 * v.double().abs().max()
    assert ((got.double().cpu() - want).abs() <= tol).all(), ((got.double().cpu() - want).abs() / want.abs()).max()
