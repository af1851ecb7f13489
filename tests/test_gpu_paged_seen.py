"""Paged attention where a batch says more than its table or ``max_seqlen`` holds."""
import pytest
import torch

import paged_reference as R
from conftest import announce

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _i(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _pages(pages, heads, page, D, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(pages, heads, page, D, generator=gen).to(DT[dtype]) for _ in range(2)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("prefix", [False, True])
@pytest.mark.parametrize("new", [3, 40])
def test_attention_past_the_table(gpu, new, prefix, dtype):
    """A query sees the keys up to its own place, whether or not the table holds the rest."""
    from deltaattention_amd import ops
    announce(f"paged attention past the table, {new} tokens, prefix={prefix} {dtype}")
    held, D = 64, 64
    k, v = _pages(10, 2, 16, D, dtype)
    table = torch.tensor([[4, 2, 7, 0], [1, 8, 3, 6]], dtype=torch.int32)
    for past in (held - new // 2 - 1, held, held + 5):  # some, one and none of the first sequence's places in the table
        lengths, cu = [past + new, new], [0, new, 2 * new]
        q = torch.randn(2 * new, 8, D, generator=torch.Generator().manual_seed(past)).to(DT[dtype])
        kv, batch = ops.PagedKV(k.cuda(), v.cuda()), ops.PagedBatch(table.cuda(), _i(lengths), cu)
        pre = ([[9, 5]], [19], [0, 2 * new]) if prefix else None
        if prefix:
            got = ops.shared_prefix_attention(q.cuda(), kv, batch, ops.PagedBatch(_i([[9, 5]]), _i([19]), pre[2]))
        else:
            got = ops.paged_attention(q.cuda(), kv, batch)
        # each token of the first sequence as if it were the last of a sequence that the table holds
        rows = [min(past + i + 1, held) for i in range(new)]
        own = R.attention(q[:new], k, v, [table[0].tolist()] * new, rows, list(range(new + 1)),
                          None if pre is None else (pre[0], pre[1], [0, new]))
        other = R.attention(q[new:], k, v, [table[1].tolist()], [new], [0, new],
                            None if pre is None else (pre[0], pre[1], [0, new]))
        for part, (want, tol) in ((got[:new], own), (got[new:], other)):
            assert ((part.double().cpu() - want).abs() <= tol).all(), past


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("most", [2, 40])
def test_tokens_before_max_seqlen(gpu, most, dtype):
    """Of a sequence with more tokens than max_seqlen the first ones are as they are without it, the others
    keep what the output held."""
    from deltaattention_amd import ops
    announce(f"paged attention, the first {most} tokens {dtype}")
    new, past = most + 5, 21
    k, v = _pages(9, 2, 16, 64, dtype)
    table = torch.randperm(9, generator=torch.Generator().manual_seed(3))[:5].to(torch.int32)[None].contiguous()
    q = torch.randn(new, 8, 64, generator=torch.Generator().manual_seed(4)).to(DT[dtype])
    out = torch.full((new, 8, 64), 3.0, dtype=DT[dtype], device="cuda")
    ops.paged_attention(q.cuda(), ops.PagedKV(k.cuda(), v.cuda()),
                        ops.PagedBatch(table.cuda(), _i([past + new]), _i([0, new]), most), out=out)
    want, tol = R.attention(q, k, v, table, [past + new], [0, new])
    assert ((out.double().cpu() - want).abs() <= tol)[:most].all()
    assert (out[most:] == 3).all()
