"""Accumulated attention weights of keys against a plain restatement in 64 bits."""
import math

import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

CASES = [  # B, H, G, D, Nq, Nk, lengths, start, anchors, dtype
    (1, 1, 1, 8, 1, 1, None, None, False, "bf16"), (1, 1, 1, 128, 1, 33, None, None, False, "bf16"),
    (2, 2, 4, 128, 5, 300, None, None, False, "bf16"), (1, 2, 4, 64, 130, 130, None, None, False, "fp16"),
    (1, 1, 7, 80, 77, 500, None, None, False, "fp16"), (1, 1, 1, 96, 300, 300, None, None, False, "fp32"),
    (2, 1, 4, 128, 64, 1000, None, None, False, "fp32"), (1, 1, 16, 40, 33, 257, [200], None, False, "bf16"),
    (1, 3, 4, 128, 33, 900, [900, 0, 1], 1500, True, "bf16"), (2, 2, 2, 64, 9, 129, [129, 128, 5, 64], 100, True, "fp32"),
    (1, 1, 64, 64, 3, 70, [70], 200, True, "fp16"), (1, 2, 4, 128, 700, 1024, None, None, False, "bf16"),
    # queries before the first keys: some see nothing
    (1, 2, 2, 64, 40, 100, None, -20, False, "bf16"), (1, 1, 3, 72, 50, 64, [64], 30, True, "fp32"),
    # queries after every key
    # a group larger than a stage of rows, of either type
    (1, 1, 64, 32, 40, 90, None, None, False, "fp32"), (1, 1, 48, 32, 40, 90, None, None, False, "fp32"),
    (1, 1, 64, 32, 40, 90, None, None, False, "bf16"), (1, 2, 3, 128, 90, 90, None, None, False, "bf16"),
    (1, 1, 4, 128, 6, 2049, None, 5000, False, "bf16"), (1, 1, 1, 128, 1, 40000, None, None, False, "bf16"),
    # one launch for both passes, and just not; few keys under many queries
    (2, 2, 4, 128, 32, 128, [128, 0, 1, 77], 200, True, "fp16"), (1, 2, 1, 96, 128, 128, None, None, False, "fp32"),
    (1, 1, 43, 128, 3, 128, [100], 150, True, "bf16"), (1, 2, 8, 64, 3000, 45, [45, 31], 20, True, "fp32"),
]


def _ids(c):
    return f"B{c[0]}H{c[1]}G{c[2]}D{c[3]}-{c[4]}x{c[5]}-{'anchors' if c[8] else 'keys'}-{c[7]}-{c[9]}"


def _want(q, k, counts, ts, lens, start):
    """(mass, bound) [B, H, N] in 64 bits."""
    B, Hq, Nq, D = q.shape
    H, N = k.shape[1], k.shape[2]
    G = Hq // H
    mass, bound = torch.zeros(B, H, N).double(), torch.zeros(B, H, N).double()
    for b in range(B):
        for h in range(H):
            n = N if lens is None else min(max(int(lens[b, h]), 0), N)
            if n == 0:
                continue
            size = torch.ones(n).double() if counts is None else counts[b, h, :n].double()
            when = torch.arange(n) if ts is None else ts[b, h, :n].long()
            kk = torch.where(size[:, None] > 0, k[b, h, :n].double(), torch.zeros(n, D).double())
            seen = (when[None] <= start + torch.arange(Nq)[:, None]) & (size > 0)[None]
            for g in range(G):
                qq = q[b, h * G + g].double()
                s = (qq @ kk.T) * D ** -0.5 + size.clamp(min=1e-300).log()
                s = torch.where(seen, s, torch.full_like(s, -math.inf))
                top = s.amax(-1, keepdim=True)
                some = torch.isfinite(top)
                w = torch.where(some, torch.exp(s - torch.where(some, top, torch.zeros_like(top))), torch.zeros_like(s))
                w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
                # fp32 scores of at most 6 D products (three parts an operand, and what they
                # leave out, 2^-23 of |q||k|), the logarithm of the sum, both exp2
                qk = (qq.abs() @ kk.abs().T).amax(-1) * D ** -0.5
                size_s = torch.where(seen, s.abs(), torch.zeros_like(s)).amax(-1)
                rel = 2.0 * ((6 * D + 4) * qk + 8 * size_s + n + 64) * 2.0 ** -24
                mass[b, h, :n] += w.sum(0)
                bound[b, h, :n] += (w * rel[:, None]).sum(0)
    return mass, bound + mass * (G * Nq + 64) * 2.0 ** -24 + 1e-35


@pytest.mark.parametrize("c", CASES, ids=[_ids(c) for c in CASES])
def test_attention_mass(gpu, c):
    from deltaattention_amd import ops
    B, H, G, D, Nq, Nk, lengths, start, anchors, dtype = c
    gen = torch.Generator().manual_seed(Nq * 7 + Nk + D)
    dt = DTYPES[dtype]
    q = (1.5 * torch.randn(B, Nq, H * G, D, generator=gen)).to(dt).transpose(1, 2)
    k = (torch.randn(B, Nk, H, D, generator=gen) * torch.exp(0.5 * torch.randn(1, 1, H, D, generator=gen))).to(dt).transpose(1, 2)
    counts = ts = lens = None
    if anchors:
        counts = torch.randint(1, 6, (B, H, Nk), generator=gen, dtype=torch.int32)
        ts = (counts.cumsum(-1) - counts).int()
        counts[torch.rand(B, H, Nk, generator=gen) < 0.1] = 0
    if lengths is not None:
        lens = torch.tensor(lengths, dtype=torch.int32).view(B, H)
    begin = Nk - Nq if start is None else start
    want, bound = _want(q, k, counts, ts, lens, begin)
    # what no query may look at: keys past the length, keys of count 0
    dead = torch.zeros(B, H, Nk, dtype=torch.bool)
    if counts is not None:
        dead |= counts <= 0
    if lens is not None:
        dead |= torch.arange(Nk) >= lens[..., None]
    k = k.clone()
    k[dead] = torch.tensor([math.nan, math.inf] * (D // 2)).to(dt)
    dev = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    announce(f"mass {_ids(c)}")
    got = ops.attention_mass(dev(q), dev(k), dev(counts), dev(ts), dev(lens), q_start=start).cpu().double()
    off = (got - want).abs()
    assert (off <= bound).all(), f"{(off / bound).max():.3g} of the bound"
    assert (got[dead] == 0).all()
    again = ops.attention_mass(dev(q), dev(k), dev(counts), dev(ts), dev(lens), q_start=start).cpu().double()
    assert torch.equal(again, got)


def test_attention_mass_blind_nan_queries(gpu):
    """Queries that see no key add nothing, whatever they hold."""
    from deltaattention_amd import ops
    gen = torch.Generator().manual_seed(9)
    q = torch.randn(1, 4, 40, 64, generator=gen).bfloat16()
    k = torch.randn(1, 2, 60, 64, generator=gen).bfloat16()
    q[:, :, :10] = math.nan
    announce("mass blind queries")
    got = ops.attention_mass(q.to(gpu), k.to(gpu), q_start=-10).cpu().double()
    want, bound = _want(q[:, :, 10:], k, None, None, None, 0)
    assert ((got - want).abs() <= bound).all()


def test_attention_mass_large_scores(gpu):
    """Scores far apart: the maximum moves by more than fp32's exponents hold."""
    from deltaattention_amd import ops
    gen = torch.Generator().manual_seed(10)
    k = torch.randn(1, 1, 500, 128, generator=gen).bfloat16()
    q = (40.0 * torch.randn(1, 2, 70, 128, generator=gen)).bfloat16()
    k[0, 0, 300] = 3 * q[0, 0, 5] / 40.0
    announce("mass large scores")
    got = ops.attention_mass(q.to(gpu), k.to(gpu), q_start=600).cpu().double()
    want, bound = _want(q, k, None, None, None, 600)
    assert ((got - want).abs() <= bound).all()
    assert abs(float(got.sum()) - 140.0) < 1e-2
