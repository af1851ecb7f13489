"""Shared prefixes: groups with more tokens than the prefix's max_seqlen says."""
import pytest
import torch

import paged_reference as R
from conftest import announce

pytestmark = pytest.mark.gpu


def _i(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new,prefix", [(1, 40), (1, 3000), (20, 200)])
def test_tokens_past_a_groups_max_seqlen(gpu, new, prefix, dtype):
    """They keep what the output held, as in a sequence: no answer without the prefix."""
    from deltaattention_amd import ops
    announce(f"shared prefix, {new} tokens a sequence, max_seqlen too small {dtype}")
    B, page, D = 9, 16, 64
    gen = torch.Generator().manual_seed(1)
    past = [3 * b for b in range(B)]
    lengths, cu = [p + new for p in past], [new * b for b in range(B + 1)]
    tables, P = R.tables(lengths + [prefix, 17], page, gen=gen)
    k, v = (torch.randn(P, 2, page, D, generator=gen).to(dtype) for _ in range(2))
    q = torch.randn(cu[-1], 8, D, generator=gen).to(dtype)
    groups, most = [new, 5 * new, 9 * new], 3 * new  # the first sequence is in none; of four in each, three count
    out = torch.full((cu[-1], 8, D), 3.0, dtype=dtype, device="cuda")
    ops.shared_prefix_attention(q.cuda(), ops.PagedKV(k.cuda(), v.cuda()), ops.PagedBatch(tables[:B].contiguous().cuda(), _i(lengths), cu),
                                ops.PagedBatch(tables[B:].contiguous().cuda(), _i([prefix, 17]), _i(groups), most), out=out)
    want, tol = R.attention(q, k, v, tables[:B], lengths, cu, (tables[B:], [prefix, 17], groups))
    for b in range(B):
        rows = slice(cu[b], cu[b + 1])
        if b in (4, 8):
            assert (out[rows] == 3).all()
        else:
            assert ((out[rows].double().cpu() - want[rows]).abs() <= tol[rows]).all()
