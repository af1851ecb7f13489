"""What a lost bf16 part would do to the 4-bit cache's attention and to the accumulated weights.

The kernels cut what does not fit bf16 into parts: q into 1 (bf16), 2 (fp16) or 3 (fp32), the softmax
weights into 2 (16-bit outputs) or 3, and for accumulated weights fp32 q and k into 3.  The worst-case
bounds of the other tests are too wide to see that one is gone, since errors of many terms rarely add up.
Here an error is a root mean square over all outputs, and its limit a third (accumulated weights: half) of
what it would be with a part less, computed in 64 bits on the same inputs.

Why a kernel with all of its parts stays under that, with x the root mean square of a relative error:
a part less leaves a value off by up to 2^-18 (two parts) or 2^-9 (one), x about 2^-19.3 or 2^-10.3 of it.
A score of about 1 (the inputs') and its weight have in fp32 about 48 additions of x 2^-25.5, the scale,
log2(count), the distance to the maximum (below 16: steps of 2^-20) and exp2 of one rounding each, in all
x about 2^-22.  The output's own rounding is x 2^-13.5 (fp16) or 2^-10.5 (bf16) of the output, as much as a
lost part of bf16's weights: there the inputs keep the output at a twelfth of the terms that it is the sum of
(the rows come in pairs with one key, opposite values and counts c and c + 1)."""
import math

import torch

PARTS = {"bf16": (1, 2), "fp16": (2, 2), "fp32": (3, 3)}  # of q, of the weights
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def cut(x, n):
    """The sum of ``n`` bf16 parts of x (float64 in and out; each part rounds what the others left)."""
    total = torch.zeros_like(x)
    for _ in range(n):
        total = total + (x - total).bfloat16().double()
    return total


def attention_inputs(B, H, G, D, rows, dtype, seed):
    """(q [B, H G, D], k, v [B, H, rows, D], counts [B, H, rows]) on the CPU, scores of about 1."""
    gen = torch.Generator().manual_seed(seed)
    each = 2 if dtype == "bf16" else 1
    some = (rows + each - 1) // each
    k, v = (torch.randn(B, H, some, D, generator=gen).repeat_interleave(each, 2)[:, :, :rows].clone() for _ in range(2))
    counts = torch.randint(8, 16, (B, H, some), generator=gen, dtype=torch.int32).repeat_interleave(each, 2)[:, :, :rows].clone()
    if each == 2:
        v[:, :, 1::2] *= -1.0
        counts[:, :, 1::2] += 1
    q = torch.randn(B, H * G, D, generator=gen).to(DTYPES[dtype])
    return q, k, v, counts


def attention(q, k, v, counts, q_parts=None, p_parts=None):
    """(out, weights summed over the group) in 64 bits; q and the weights cut where asked."""
    B, H, n, D = k.shape
    qq = q.double() if q_parts is None else cut(q.double(), q_parts)
    s = torch.matmul(qq.view(B, H, -1, D), k.double().transpose(-1, -2).contiguous()) * D ** -0.5
    w = torch.exp(s - s.amax(-1, keepdim=True)) * counts.double()[:, :, None]
    L = w.sum(-1, keepdim=True)
    out = torch.matmul(w if p_parts is None else cut(w, p_parts), v.double()) / L
    return out.view(q.shape), (w / L).sum(2)


def emulate(q, k, v, counts, dtype, q_parts, p_parts):
    """The kernels' arithmetic in fp32 on the CPU, with these numbers of parts."""
    B, H, n, D = k.shape
    qq, kt = q.double().view(B, H, -1, D), k.transpose(-1, -2).contiguous()
    s, left = 0.0, qq
    for _ in range(q_parts):
        part = left.bfloat16()
        left = left - part.double()
        s = s + torch.matmul(part.float(), kt)
    s = s * torch.tensor(D ** -0.5 * math.log2(math.e)) + torch.log2(counts.float())[:, :, None]
    w = torch.exp2(s - s.amax(-1, keepdim=True))
    L = w.sum(-1, keepdim=True)
    o, rest = 0.0, w
    for _ in range(p_parts):
        part = rest.bfloat16().float()
        rest = rest - part
        o = o + torch.matmul(part, v)
    return (o / L).view(q.shape).to(DTYPES[dtype]), (w / L).sum(2)


def _rms(x):
    return float(x.double().pow(2).mean().sqrt())


def attention_ratios(out, mass, q, k, v, counts, dtype):
    """Errors over those of a lost part: (out, q one part less), (out, weights one less), (mass, q one less).
    None where there is no part to lose."""
    q_parts, p_parts = PARTS[dtype]
    want, weights = attention(q, k, v, counts)
    err, merr = _rms(out.double() - want), None if mass is None else _rms(mass.double() - weights)
    lost_q = lost_m = None
    if q_parts > 1:
        less, less_w = attention(q, k, v, counts, q_parts=q_parts - 1)
        lost_q = err / _rms(less - want)
        lost_m = None if merr is None else merr / _rms(less_w - weights)
    lost_p = err / _rms(attention(q, k, v, counts, p_parts=p_parts - 1)[0] - want)
    return lost_q, lost_p, lost_m


def assert_attention(out, mass, q, k, v, counts, dtype):
    for what, ratio in zip(("a part of q (out)", "a part of the weights", "a part of q (mass)"),
                           attention_ratios(out, mass, q, k, v, counts, dtype)):
        assert ratio is None or ratio < 1 / 3, f"{ratio:.3f} of the error without {what}"


def mass_inputs(B, H, G, D, Nq, Nk, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(B, H * G, Nq, D, generator=gen), torch.randn(B, H, Nk, D, generator=gen)


def mass(q, k, parts=(None, None)):
    """Accumulated weights in 64 bits of queries that see every key, q and k cut where asked."""
    B, H, n, D = k.shape
    qq, kk = (x.double() if p is None else cut(x.double(), p) for x, p in zip((q, k), parts))
    s = torch.matmul(qq.view(B, H, -1, D), kk.transpose(-1, -2).contiguous()) * D ** -0.5
    return torch.softmax(s, -1).sum(2)


def assert_mass(got, q, k):
    want = mass(q, k)
    err = _rms(got.double() - want)
    for what, parts in (("q", (2, None)), ("k", (None, 2))):
        ratio = err / _rms(mass(q, k, parts) - want)
        assert ratio < 1 / 2, f"{ratio:.3f} of the error without a part of {what}"


def emulate_mass(q, k, products):
    """The kernels' arithmetic in fp32 on the CPU: the products (part of q, part of k) that are kept."""
    B, H, n, D = k.shape

    def parts(x):
        got = []
        for _ in range(3):
            got.append(x.bfloat16().float())
            x = x - got[-1]
        return got
    qs, ks = parts(q.view(B, H, -1, D)), parts(k)
    s = 0.0
    for i, j in products:
        s = s + torch.matmul(qs[i], ks[j].transpose(-1, -2).contiguous())
    s = s * torch.tensor(D ** -0.5 * math.log2(math.e))
    w = torch.exp2(s - s.amax(-1, keepdim=True))
    return (w / w.sum(-1, keepdim=True)).sum(2)
