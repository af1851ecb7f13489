"""The paged cache's operators where cu_seqlens does not rise: no place outside the batch is read or written."""
import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu


def _i(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


CUS = [[0, 1000, 20, 43], [0, 30, 2, 43], [43, 30, 10, 0], [-7, 20, -3, 50], [5, 5, 4, 40], [0, 0, 1 << 30, -(1 << 31)]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("prefix", [0, 40, 3000])
@pytest.mark.parametrize("cu", CUS)
def test_attention_stays_inside(gpu, cu, prefix, dtype):
    """Outputs beside the batch's keep what they held, and the next call is as it should be."""
    from deltaattention_amd import ops
    announce(f"paged attention, cu {cu}, prefix of {prefix} {dtype}")
    T, page, lengths, wide = 43, 16, [50, 20, 48], 64
    kv = ops.PagedKV(*(torch.randn(wide * 4, 2, page, 64, device="cuda").to(dtype) for _ in range(2)))
    table = torch.randperm(wide * 4, device="cuda").to(torch.int32).view(4, wide)
    q = torch.randn(T, 8, 64, device="cuda").to(dtype)
    good = ops.PagedBatch(table[:3], _i(lengths), [0, 1, 20, 43])

    def call(batch, order, out=None):
        if not prefix:
            return ops.paged_attention(q, kv, batch, out=out)
        pre = ops.PagedBatch(table[3:].repeat(3, 1), _i([min(prefix, wide * page)] * 3), _i(order), 43)
        return ops.shared_prefix_attention(q, kv, batch, pre, out=out)
    want = call(good, [0, 1, 20, 43])
    assert torch.isfinite(want).all()
    whole = torch.full((T + 8, 8, 64), 3.0, dtype=dtype, device="cuda")
    for most in (1, 5, 43):
        call(ops.PagedBatch(table[:3], _i(lengths), _i(cu), most), cu, whole[4:T + 4])
        assert (whole[:4] == 3).all() and (whole[T + 4:] == 3).all()
        assert torch.equal(call(good, [0, 1, 20, 43]), want)
