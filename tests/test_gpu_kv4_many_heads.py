"""Decode attention over 4-bit rows for many (sequence, KV head) pairs: around the numbers of pairs and
of rows where the call's form changes, every head against the definition in 64 bits."""
import math

import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)

CASES = [  # B, H, G, D, capacity, W, dtype
    (32, 8, 4, 8, 1000, 5, "bf16"), (16, 16, 16, 40, 1024, 3, "fp16"), (52, 5, 4, 8, 1025, 1, "bf16"),
    (16, 16, 17, 8, 1000, 2, "bf16"), (96, 8, 16, 8, 1024, 4, "bf16"), (96, 8, 16, 8, 1100, 4, "bf16"),
    (96, 8, 8, 8, 2100, 4, "fp16"), (96, 8, 4, 8, 4200, 4, "bf16"), (97, 8, 4, 8, 4225, 17, "fp32"),
    (95, 8, 4, 8, 4200, 4, "bf16"), (800, 1, 1, 8, 17000, 2, "bf16"), (768, 1, 40, 8, 1100, 2, "fp32"),
]


def _ids(c):
    return f"B{c[0]}H{c[1]}G{c[2]}D{c[3]}-cap{c[4]}-{c[6]}"


def _values(codes, scales, D):
    """The values of 4-bit rows, float64."""
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float64, device=codes.device)
    x = level[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()]
    return x[..., :D] * torch.pow(2.0, scales.double() - 127.0).repeat_interleave(32, -1)[..., :D]


@pytest.mark.parametrize("c", CASES, ids=[_ids(c) for c in CASES])
def test_attend_many_heads(gpu, c):
    from deltaattention_amd import ops
    B, H, G, D, cap, W, dtype = c
    dt, groups = DTYPES[dtype], (D + 31) // 32
    gen = torch.Generator(device=gpu).manual_seed(B + H + cap)
    new = lambda *s, lo, hi, t: torch.randint(lo, hi, s, generator=gen, device=gpu).to(t)  # noqa: E731
    codes = [new(B, H, cap, 16 * groups, lo=0, hi=256, t=torch.uint8) for _ in range(2)]
    for x in codes:
        x.view(B, H, cap, -1)[..., (D + 1) // 2:] = 0  # dims past the head's
    scales = [new(B, H, cap, groups, lo=123, hi=127, t=torch.uint8) for _ in range(2)]
    counts = new(B, H, cap, lo=0, hi=9, t=torch.int32)
    lengths = new(B, H, lo=cap // 2, hi=cap + 1, t=torch.int32)
    lengths[0, 0], lengths[-1, -1], lengths[B // 2, 0] = cap, cap, 0
    start = torch.rand(B, H, cap, generator=gen, device=gpu)
    kv = ops.KV4(codes[0], scales[0], codes[1], scales[1], counts, torch.zeros_like(counts), lengths, D, start.clone())
    q = torch.randn(B, H * G, 1, D, generator=gen, device=gpu).to(dt)
    kx, vx = (torch.randn(B, H, W, D, generator=gen, device=gpu).to(dt) for _ in range(2))
    announce(f"attend many heads {_ids(c)}")
    out = ops.decode_attention_kv4(q, kv, kx, vx)
    assert torch.equal(kv.mass, start)
    both = ops.decode_attention_kv4(q, kv, kx, vx, accumulate=True)
    torch.cuda.synchronize()
    for b0 in range(0, B, 96):  # a part of the batch at a time: the 64-bit values are wide
        sl = slice(b0, min(b0 + 96, B))
        n = min(96, B - b0) * H
        k = torch.cat([_values(codes[0][sl], scales[0][sl], D), kx[sl].double()], 2).view(n, cap + W, D)
        v = torch.cat([_values(codes[1][sl], scales[1][sl], D), vx[sl].double()], 2).view(n, cap + W, D)
        size = torch.cat([counts[sl].double(), torch.ones(counts[sl].shape[0], H, W, device=gpu).double()], 2).view(n, 1, -1)
        row = torch.arange(cap + W, device=gpu)
        live = (size > 0) & ((row >= cap) | (row < lengths[sl].reshape(n, 1, 1)))
        qq = q[sl].double().view(n, G, D)
        kt = k.transpose(1, 2).contiguous()
        s = torch.matmul(qq, kt) * D ** -0.5 + torch.where(live, size, torch.ones_like(size)).log()
        s = torch.where(live, s, torch.full_like(s, -math.inf))
        p = torch.softmax(s, -1)
        want = torch.matmul(p, v)
        spread = torch.matmul(p, v.abs())
        # a score: at most 6 D products rounded and added in fp32, then scale, log2 and log(count) of one
        # rounding each, the maximum's difference and exp2 likewise; a weight's parts leave 2^-17 (16-bit
        # outputs) or less, sums have cap + W terms; the output's own rounding is half a step
        size_qk = (torch.matmul(qq.abs(), kt.abs()) * live).amax(-1, keepdim=True) * D ** -0.5
        drift = 2.0 * (6 * D * size_qk + 8 * torch.where(live, s, torch.zeros_like(s)).abs().amax(-1, keepdim=True) + 8) * 2.0 ** -24
        eps = torch.finfo(dt).eps / 2
        rel = drift + 2.0 ** -16 * (dtype != "fp32") + (cap + W + 64) * 2.0 ** -24
        tol = eps * want.abs() + (1 + eps) * rel * spread + 1e-30
        for got in (out, both):
            off = (got[sl].double().view(n, G, D) - want).abs()
            assert (off <= tol).all(), f"{(off / tol).max():.3g} of the bound"
        add = p[..., :cap].sum(1).view(-1, H, cap)
        wtol = (p[..., :cap] * (drift + (cap + W + 64) * 2.0 ** -24)).sum(1).view(-1, H, cap) + 2.0 ** -23 * (add + start[sl].double())
        off = (kv.mass[sl].double() - start[sl].double() - add).abs()
        used = torch.arange(cap, device=gpu) < lengths[sl][..., None]
        assert (off <= wtol)[used].all(), f"weights {(off / wtol)[used].max():.3g} of the bound"
        assert torch.equal(kv.mass[sl][~used], start[sl][~used])  # rows behind the length stay
