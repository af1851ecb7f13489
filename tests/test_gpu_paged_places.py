"""Writing into the paged cache: every token to its own place or to none."""
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


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lengths,cu,most", [
    ([33], [0, 2], 2),             # the second token is past a table of 32 rows
    ([34], [0, 2], 2),             # both are
    ([1 << 30], [0, 2], 2),
    ([30], [0, 9], 4),             # more tokens than max_seqlen says
    ([40, 20], [0, 12, 15], 5),    # both at once, beside a sequence as it should be
])
def test_append_past_the_table(gpu, lengths, cu, most, dtype):
    """A token's place is its own: past the table it is dropped, and no row before it is touched."""
    from deltaattention_amd import ops
    announce(f"append past the table {lengths} {cu} {most} {dtype}")
    B, T = len(lengths), cu[-1]
    k, v = _pages(2 * B + 1, 2, 16, 64, dtype)
    table = torch.arange(2 * B, dtype=torch.int32).view(B, 2).flip(1).contiguous()
    gen = torch.Generator().manual_seed(1)
    new_k, new_v, q = (torch.randn(T, h, 64, generator=gen).to(DT[dtype]) for h in (2, 2, 4))
    angle = torch.arange(50.0, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(32).double() / 32)
    cos, sin = angle.cos().float(), angle.sin().float()
    place = [(b, lengths[b] - cu[b + 1] + t) for b in range(B) for t in range(cu[b], cu[b + 1])]
    at = torch.tensor([min(max(slot, 0), 49) for _, slot in place])
    turned, tol = R.rotate(new_k, cos[at], sin[at], False)
    want_k, want_v, tol_k = k.double(), v.double(), torch.zeros(k.shape, dtype=torch.float64)
    for t, (b, slot) in enumerate(place):
        if 0 <= slot < 32:
            page, row = int(table[b, slot // 16]), slot % 16
            want_k[page, :, row], tol_k[page, :, row], want_v[page, :, row] = turned[t], tol[t], new_v[t].double()
    kv = ops.PagedKV(k.cuda(), v.cuda())
    got = ops.append_paged(kv, ops.PagedBatch(table.cuda(), _i(lengths), _i(cu), most), new_k.cuda(), new_v.cuda(),
                           q=q.cuda(), cos=cos.cuda(), sin=sin.cuda())
    assert ((kv.k_pages.double().cpu() - want_k).abs() <= tol_k).all()
    assert torch.equal(kv.v_pages.double().cpu(), want_v)
    turned, tol = R.rotate(q, cos[at], sin[at], False)
    assert ((got.double().cpu() - turned).abs() <= tol).all()


def places(lengths, cu, T, table, page):
    """The (page, row) places that tokens of a batch may be written to: token t of sequence b, of those that
    cu[b] <= t < cu[b + 1], to slot lengths[b] - cu[b + 1] + t of its table."""
    out = set()
    for b, row in enumerate(table):
        for t in range(max(cu[b], 0), min(cu[b + 1], T)):
            slot = lengths[b] - cu[b + 1] + t
            if 0 <= slot < len(row) * page and row[slot // page] >= 0:
                out.add((row[slot // page], slot % page))
    return out


CUS = [[0, 1000, 20, 43], [0, 30, 2, 43], [43, 30, 10, 0], [-7, 20, -3, 50], [5, 5, 4, 40], [0, 0, 1 << 30, -(1 << 31)]]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("cu", CUS)
def test_append_writes_its_places_only(gpu, cu, dtype):
    from deltaattention_amd import ops
    announce(f"append, cu {cu} {dtype}")
    T, page, lengths = 43, 16, [50, 20, 48]
    whole = [torch.randn(14, 2, page, 64, device="cuda").to(DT[dtype]) for _ in range(2)]
    kv = ops.PagedKV(*(x[1:13] for x in whole))  # pages before and behind that belong to others
    table = [[3, 11, 0, 7], [1, 9, 2, 8], [6, 4, 10, 5]]
    before = [x.clone() for x in whole]
    x = torch.full((T, 2, 64), 5.0, dtype=DT[dtype], device="cuda")
    ops.append_paged(kv, ops.PagedBatch(_i(table), _i(lengths), _i(cu), 43), x, x)
    may = places(lengths, cu, T, table, page)
    for now, old in zip(whole, before):
        changed = {(int(p) - 1, int(r)) for p, r in (now != old).any(-1).any(1).nonzero()}
        assert changed <= may, sorted(changed - may)
