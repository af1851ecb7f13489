"""Paged attention of few rows: long shares of the key stream, and what other sequences may change."""
import pytest
import torch

import paged_reference as R
from conftest import announce

pytestmark = pytest.mark.gpu


def _i(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths", [[80011, 75003, 84977, 79900], [134001, 140123, 90007, 195511]])
def test_shares_of_many_tiles(gpu, lengths, dtype):
    """Workers with more than 32 and more than 64 tiles of one item, which begin in its middle: the numbers of a
    run's pages are read 32 tiles at a time."""
    from deltaattention_amd import ops
    announce(f"paged decode of {lengths} {dtype}")
    Hkv, D, page, G = 8, 64, 16, 4
    tiles = Hkv * sum(-(-n // 128) for n in lengths)
    workers = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    assert -(-tiles // workers) > (32 if lengths[0] < 100000 else 64)
    gen = torch.Generator(device="cuda").manual_seed(2)
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(need) + 5, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((4, max(need)), -1, dtype=torch.int32, device="cuda")
    for b, m in enumerate(need):
        table[b, :m] = order[sum(need[:b]):sum(need[:b]) + m]
    k, v = (torch.randn(sum(need) + 5, Hkv, page, D, generator=gen, device="cuda").to(dtype) for _ in range(2))
    q = (2.0 * torch.randn(4, Hkv * G, D, generator=gen, device="cuda")).to(dtype)
    got = ops.paged_attention(q, ops.PagedKV(k, v), ops.PagedBatch(table, _i(lengths)))
    assert torch.isfinite(got).all()
    for b, h in ((0, 0), (1, 3), (2, 7), (3, 5), (3, 7)):
        rows = [x[table[b, :need[b]].long(), h].reshape(1, 1, -1, D)[:, :, :lengths[b]].cpu() for x in (k, v)]
        whole = [torch.cat([x, torch.zeros(1, 1, -x.shape[2] % page, D, dtype=dtype)], 2).view(1, -1, page, D).transpose(0, 1)
                 for x in rows]
        one = q[b:b + 1, h * G:(h + 1) * G].cpu()
        want, tol = R.attention(one, *whole, [list(range(need[b]))], [lengths[b]], [0, 1])
        assert ((got[b:b + 1, h * G:(h + 1) * G].double().cpu() - want).abs() <= tol).all(), (b, h)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("new", [[1, 33, 1, 1], [1, 1, 1, 1], [200, 1, 40, 3]])
def test_companions(gpu, new, dtype):
    """What other sequences hold changes no bit of a sequence's result; how long they are may change the order of
    its sums, within the bound."""
    from deltaattention_amd import ops
    announce(f"paged attention beside others {new} {dtype}")
    past, page, D = [5000, 200, 31, 2222], 16, 128
    cu = [sum(new[:b]) for b in range(5)]
    gen = torch.Generator().manual_seed(6)
    lengths = [n + p for n, p in zip(new, past)]
    table, P = R.tables([n + 3000 for n in lengths], page, gen=gen)
    k, v = (torch.randn(P, 2, page, D, generator=gen).to(dtype) for _ in range(2))
    q = torch.randn(cu[-1], 8, D, generator=gen).to(dtype)

    def call(k, v, q, lengths):
        return ops.paged_attention(q.cuda(), ops.PagedKV(k.cuda(), v.cuda()), ops.PagedBatch(table.cuda(), _i(lengths), cu)).cpu()
    first = call(k, v, q, lengths)
    for b in range(4):
        mine = torch.zeros(P, dtype=torch.bool)
        mine[table[b][table[b] >= 0].long()] = True
        other = [torch.where(mine[:, None, None, None], x, torch.full_like(x, float("nan"))) for x in (k, v)]
        rest = torch.full_like(q, float("nan"))
        rest[cu[b]:cu[b + 1]] = q[cu[b]:cu[b + 1]]
        assert torch.equal(call(*other, rest, lengths)[cu[b]:cu[b + 1]], first[cu[b]:cu[b + 1]])
        longer = [n if i == b else n + 3000 - 700 * i for i, n in enumerate(lengths)]
        got = call(k, v, q, longer)[cu[b]:cu[b + 1]]
        want, tol = R.attention(q[cu[b]:cu[b + 1]], k, v, [table[b].tolist()], [lengths[b]], [0, new[b]])
        assert ((got.double() - want).abs() <= tol).all()
