"""Row choice where accumulated weights hold NaN: a NaN of either sign and any payload is the largest,
all of them tie, and ties go to the lower row."""
import math

import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu

# bit patterns: quiet and signalling NaN, both signs, the smallest and largest payloads
NANS = (0x7FC00000, 0xFFC00000, 0x7F800001, 0xFF800001, 0x7FFFFFFF, 0xFFFFFFFF)


def _mass(gen, shape, share):
    pool = torch.tensor([0.0, -0.0, 1.0, -1.0, math.inf, -math.inf, 3e38, 1e-45], dtype=torch.float32).view(torch.int32)
    bits = pool[torch.randint(0, len(pool), shape, generator=gen)]
    nans = torch.tensor([x - (1 << 32) if x >> 31 else x for x in NANS], dtype=torch.int32)
    odd = nans[torch.randint(0, len(nans), shape, generator=gen)]
    return torch.where(torch.rand(shape, generator=gen) < share, odd, bits).view(torch.float32)


def _rows(mass, n, budget, sinks, recent):
    if n <= budget:
        return list(range(n))
    key = [(0, 0.0) if math.isnan(m) else (1, -m) for m in mass.tolist()]
    middle = sorted(range(sinks, n - recent), key=lambda j: (key[j], j))[:budget - sinks - recent]
    return sorted(list(range(sinks)) + middle + list(range(n - recent, n)))


@pytest.mark.parametrize("share", [0.01, 0.3, 1.0])
@pytest.mark.parametrize("N,lengths,budget,sinks,recent", [
    (90, [90, 89, 40, 12], 40, 2, 8), (3000, [3000, 2999, 1000, 0], 700, 4, 64), (20000, [20000, 17001, 300, 9000], 8000, 0, 1),
    (20000, [20000, 19999, 17000, 64], 50, 16, 2)])
def test_nan_is_the_largest(gpu, N, lengths, budget, sinks, recent, share):
    from deltaattention_amd import ops
    gen = torch.Generator().manual_seed(N + budget)
    mass = _mass(gen, (2, 2, N), share)
    lens = torch.tensor(lengths, dtype=torch.int32).view(2, 2)
    announce(f"heavy nan N={N} budget={budget} share={share}")
    kv = ops.KV4.empty(2, 2, N, 8, gpu)
    for t in (kv.k_codes, kv.k_scales, kv.v_codes, kv.v_scales, kv.counts):
        t.zero_()
    kv.timestamps.copy_(torch.arange(N, dtype=torch.int32).expand(2, 2, N))
    kv.lengths.copy_(lens)
    kv.mass.view(torch.int32).copy_(mass.view(torch.int32))  # the bits as they are
    index, kept = ops.heavy_rows(kv.mass, budget, sinks, recent, lengths=kv.lengths)
    small = ops.evict_kv4(kv, budget, sinks, recent)
    for b in range(2):
        for h in range(2):
            want = _rows(mass[b, h], int(lens[b, h]), budget, sinks, recent)
            assert int(kept[b, h]) == len(want) == int(small.lengths[b, h])
            assert index[b, h].tolist() == want + [-1] * (budget - len(want))
            assert small.timestamps[b, h, :len(want)].tolist() == want
            got = small.mass[b, h, :len(want)].view(torch.int32).cpu()
            assert torch.equal(got, mass[b, h].view(torch.int32)[want])
