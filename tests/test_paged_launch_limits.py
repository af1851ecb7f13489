"""Calls of the paged cache's operators that are larger than one launch may be."""
import pytest
import torch

from deltaattention_amd import _native
from test_paged_refusals import A, BF16, _append, _batch, _kv, _refused


def test_append_of_too_many_tokens():
    """A wave a token: 2^26 of them are 2^32 threads."""
    for T in (1 << 26, 1 << 28, 1 << 40):
        _refused(_append(T=T), -1, "2^26 tokens")


def _workspace(B):
    return _native.lib().da_paged_attention_workspace_size(BF16, B, 8, 8, 8, _kv(), _batch(cu=None, B=B, width=1, table_stride=1),
                                                           None)


def test_decode_of_millions_of_items():
    """Short caches take a workgroup a sequence and head and no workspace; 2^24 of those are 2^32 threads, so they
    go in equal shares as long ones do, through a workspace."""
    assert _workspace((1 << 21) - 1) == 0
    assert _workspace(1 << 21) > 0
    assert A  # (addresses are not followed)


@pytest.mark.gpu
def test_decode_of_millions_of_items_on_the_gpu(gpu):
    """2^21 sequences of 8 heads, of 1 to 16 keys of one page."""
    from conftest import announce

    import paged_reference as R
    from deltaattention_amd import ops
    announce("paged decode of 2^21 sequences")
    B, gen = 1 << 21, torch.Generator().manual_seed(0)
    k, v = (torch.randn(2, 8, 16, 8, generator=gen).bfloat16() for _ in range(2))
    q = torch.randn(1, 8, 8, generator=gen).bfloat16()
    lengths = (torch.arange(B, device="cuda") % 16 + 1).to(torch.int32)
    batch = ops.PagedBatch(torch.ones(B, 1, dtype=torch.int32, device="cuda"), lengths)
    got = ops.paged_attention(q.cuda().expand(B, 8, 8), ops.PagedKV(k.cuda(), v.cuda()), batch)
    want, tol = R.attention(q.expand(16, 8, 8), k, v, [[1]] * 16, list(range(1, 17)), list(range(17)))
    assert ((got[:16].double().cpu() - want).abs() <= tol).all()
    assert torch.equal(got.view(-1, 16, 8, 8), got[:16].expand(B // 16, 16, 8, 8))
