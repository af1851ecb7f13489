"""Plain 64-bit definitions of the paged cache's operators, on the CPU, and the error bounds that
their kernels' arithmetic gives.  Test infrastructure."""
import math

import torch

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}


def rows_of(pages, table, n):
    """The first n rows of the pages that ``table`` (a list) names: [Hkv, n, D] float64; a page that is
    not there counts as zeros."""
    P, H, S, D = pages.shape
    out = torch.zeros(H, n, D, dtype=torch.float64)
    for j in range(-(-n // S)):
        page = int(table[j])
        m = min(S, n - j * S)
        if 0 <= page < P:
            out[:, j * S:j * S + m] = pages[page, :, :m].double()
    return out


def attention(q, k_pages, v_pages, table, lengths, cu, prefix=None, scale=None):
    """(out, tolerance) [T, Hq, D] float64.  ``prefix``: (table, lengths, cu over tokens).  Rows that
    belong to no sequence are NaN in both.

    The tolerance holds what the kernels may do: one rounding of the output and one of the
    weights to the tensors' type (none to fp32's own sums), scores, sums and products in fp32 in any
    order.  With w the exact weights and A = sum w |v|: weights off by a relative
    e = (D + 4) 2^-24 scale sum |q k| + 2^-23 |score| + 2^-22 from the scores and exponentials, sums of n
    terms by n 2^-24, so |out - exact| <= u |out| + (2 e + u_p + 2 n 2^-24) A."""
    T, Hq, D = q.shape
    Hkv = k_pages.shape[1]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    u = HALF_STEP[q.dtype]
    u_p = 0.0 if q.dtype == torch.float32 else u
    out = torch.full((T, Hq, D), math.nan, dtype=torch.float64)
    tol = torch.full((T, Hq, D), math.nan, dtype=torch.float64)
    for b in range(len(lengths)):
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        k, v, common = rows_of(k_pages, table[b], lengths[b]), rows_of(v_pages, table[b], lengths[b]), 0
        if prefix is not None:
            ptable, plen, pcu = prefix
            g = next((i for i in range(len(plen)) if pcu[i] <= cu[b] < pcu[i + 1]), None)
            if g is not None:
                common = plen[g]
                k = torch.cat([rows_of(k_pages, ptable[g], common), k], 1)
                v = torch.cat([rows_of(v_pages, ptable[g], common), v], 1)
        N = k.shape[1]
        x = q[cu[b]:cu[b + 1]].double().view(n, Hkv, G, D).permute(1, 2, 0, 3)  # [Hkv, G, n, D]
        s = torch.matmul(x, k.transpose(-1, -2)[:, None]) * scale
        size = torch.matmul(x.abs(), k.abs().transpose(-1, -2)[:, None]) * scale
        last = common + lengths[b] - n + torch.arange(n)
        hidden = torch.arange(N)[None] > last[:, None]
        s = s.masked_fill(hidden, -math.inf)
        top = s.amax(-1, keepdim=True) if N else s.new_zeros(s.shape[:-1] + (1,))
        top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
        w = torch.exp(s - top)
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total > 0, total, torch.ones_like(total))
        o = torch.matmul(w, v[:, None])
        e = (D + 4) * 2.0 ** -24 * size + 2.0 ** -23 * (s - top).abs().nan_to_num(posinf=0.0) + 2.0 ** -22
        e = torch.where(hidden, torch.zeros_like(e), e)
        A = torch.matmul(w * (2 * e + u_p + 2 * N * 2.0 ** -24), v.abs()[:, None])
        # the largest relative error also scales the sum that divides
        worst = (w * e).sum(-1, keepdim=True)
        t = u * o.abs() + A + worst * torch.matmul(w, v.abs()[:, None])
        out[cu[b]:cu[b + 1]] = o.permute(2, 0, 1, 3).reshape(n, Hq, D)
        tol[cu[b]:cu[b + 1]] = t.permute(2, 0, 1, 3).reshape(n, Hq, D)
    tiny = 2.0 ** -24 if q.dtype == torch.float16 else 2.0 ** -126  # below the normal numbers
    return out, tol + tiny


def rotate(x, cos, sin, interleaved):
    """(rotated, tolerance) of x [T, H, D] by cos, sin [T, R / 2]: three fp32 roundings of parts no larger
    than |x cos| + |y sin|, and the output's."""
    out = x.double().clone()
    tol = torch.zeros_like(out)
    half = cos.shape[1]
    u = HALF_STEP[x.dtype]
    d = torch.arange(half)
    one, two = (2 * d, 2 * d + 1) if interleaved else (d, d + half)
    a, b = out[..., one].clone(), out[..., two].clone()
    c, s = cos.double()[:, None], sin.double()[:, None]
    out[..., one], out[..., two] = a * c - b * s, b * c + a * s
    tol[..., one] = u * out[..., one].abs() + 3 * 2.0 ** -24 * (1 + u) * ((a * c).abs() + (b * s).abs())
    tol[..., two] = u * out[..., two].abs() + 3 * 2.0 ** -24 * (1 + u) * ((b * c).abs() + (a * s).abs())
    tiny = 2.0 ** -24 if x.dtype == torch.float16 else 2.0 ** -126
    return out, torch.where(tol > 0, tol + tiny, tol)


def tables(counts, page, spare=3, width=None, gen=None):
    """(table [B, width] int32 with -1 past a sequence's pages, pages in all), pages in random order."""
    need = [-(-n // page) for n in counts]
    total = sum(need) + spare
    order = torch.randperm(total, generator=gen).tolist()
    width = max(max(need), 1) if width is None else width
    table = torch.full((len(counts), width), -1, dtype=torch.int32)
    for b, m in enumerate(need):
        for j in range(m):
            table[b, j] = order.pop()
    return table, total
