"""The bounded decode cache's operators (deltaattention_amd/kv4.py) restated plainly in 64 bits,
on the CPU or the GPU: the 4-bit format from its definition, the row choice, the attention and
the accumulated weights.  Tolerances are returned with the values: each is a bound that follows
from the arithmetic, not from a run."""
import math

import torch

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def groups(D):
    return (D + 31) // 32


def encode(rows):
    """Rows [..., D] (any float type) -> (codes [..., 16 groups] uint8, exponents [..., groups] uint8)."""
    D = rows.shape[-1]
    x = torch.nn.functional.pad(rows.double().cpu(), (0, -D % 32)).unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad[..., None], torch.zeros_like(x), x)
    top = x.abs().amax(-1)
    e = torch.full(top.shape, -125, dtype=torch.int64)
    for _ in range(251):  # the smallest exponent for which no element exceeds 6
        e = torch.where((top > 6.0 * torch.pow(2.0, e.double())) & (e < 125), e + 1, e)
    y = x.abs() / torch.pow(2.0, e.double())[..., None]
    dist = (y[..., None] - LEVELS).abs()
    near = dist.amin(-1, keepdim=True)
    hit = dist == near  # one level, or two at a tie: then the even code
    first = hit.int().argmax(-1)
    two = hit.sum(-1) == 2
    code = torch.where(two & (first % 2 == 1), first + 1, first)
    code = code | (torch.signbit(x).to(torch.int64) << 3)
    code = torch.where(bad[..., None], torch.zeros_like(code), code).flatten(-2)
    pairs = code.unflatten(-1, (-1, 2))
    scales = torch.where(bad, torch.full_like(e, 255), e + 127)
    return (pairs[..., 0] | (pairs[..., 1] << 4)).to(torch.uint8), scales.to(torch.uint8)


def decode(codes, scales, D):
    """The values, float64 (NaN in groups marked 255)."""
    codes, scales = codes.cpu().long(), scales.cpu().double()
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    v = LEVELS[c & 7] * torch.where(c >= 8, -1.0, 1.0)
    power = torch.where(scales == 255, torch.full_like(scales, math.nan), torch.pow(2.0, scales - 127.0))
    return (v.unflatten(-1, (-1, 32)) * power[..., None]).flatten(-2)[..., :D]


def heavy(mass, n, budget, sinks, recent):
    """Rows kept of one head: mass a list of floats."""
    if n <= budget:
        return list(range(n))
    middle = sorted(range(sinks, n - recent), key=lambda j: (-mass[j], j))[:budget - sinks - recent]
    return sorted(list(range(sinks)) + middle + list(range(n - recent, n)))


def attention(q, k, v, size):
    """One head group: q [G, D], k, v [n, D], size [n] (0: no weight), all float64 -> (out [G, D],
    weights [G, n], spread [G, D] = sum p |v|, drift [G]: a bound of the relative error that fp32
    scores put on a weight)."""
    G, D = q.shape
    live = size > 0
    if not bool(live.any()):
        return torch.zeros(G, D).double(), torch.zeros(G, len(size)).double(), torch.zeros(G, D).double(), torch.zeros(G).double()
    k, v = torch.where(live[:, None], k, torch.zeros_like(k)), torch.where(live[:, None], v, torch.zeros_like(v))
    scale = D ** -0.5
    s = (q @ k.T) * scale + torch.where(live, size, torch.ones_like(size)).log()
    s = torch.where(live, s, torch.full_like(s, -math.inf))
    w = torch.exp(s - s.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    # a score: at most 6 D products rounded and added in fp32 (three parts of q), then scale,
    # log2 and log(count) of one rounding each; the maximum's difference and exp2 likewise
    size_qk = (q.abs() @ k.abs().T).amax(-1) * scale
    top = s[:, live].abs().amax(-1)
    drift = 2.0 * (6 * D * size_qk + 8 * top + 8) * 2.0 ** -24
    return w @ v, w, w @ v.abs(), drift
