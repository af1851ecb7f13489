"""Cases of the four operators that bound a decode cache: how much attention each key received,
which rows to keep for it, rows held in 4 bits, and attention over them.

A case is a dict of plain values.  Its ``op`` names the operator:

* ``mass``      ``ops.attention_mass``: the attention weight that every key received from a
  run of queries, summed over the queries and the query heads of its group;
* ``quantize``  ``ops.quantize_kv4`` and ``ops.dequantize_kv4``: key and value rows (all of them,
  or those that an index names) into a 4-bit cache and back;
* ``evict``     ``ops.evict_kv4``: the rows of most accumulated weight moved to a smaller cache;
* ``attend``    ``ops.decode_attention_kv4``: one decode token over a 4-bit cache and a ring of
  exact rows, with or without its weights added to the accumulated ones.

The 4-bit format: 32 consecutive dims of a row are a group with one power of two; an element is
sign, two exponent bits and one mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6) times that power.  The
power is the smallest for which no element of the group exceeds 6 (exponents from -125 to 125),
and elements round to nearest, ties to the even code.  Byte i of a row holds dims 2i (low half)
and 2i + 1; dims past the head dimension are zero.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ELEMENT = {"bf16": 2, "fp16": 2, "fp32": 4}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # the last 64 queries of a 32K prompt judge its keys (the project's 32-head layer)
        dict(name="mass_window_32k", op="mass", B=1, Hkv=8, G=4, D=128, Nq=64, Nk=32768, anchors=False, dtype="bf16"),
        # every query of an ordinary prompt judges the keys before it: the largest work here
        dict(name="mass_prompt_8k", op="mass", B=1, Hkv=8, G=4, D=128, Nq=8192, Nk=8192, anchors=False, dtype="bf16"),
        # a few queries over packed anchors of two sequences (counts, timestamps, ragged heads)
        dict(name="mass_anchors", op="mass", B=2, Hkv=8, G=1, D=64, Nq=33, Nk=2087, anchors=True, dtype="fp16"),
        # hand-off of a long prompt's rows to the 4-bit cache, as the projections lay them out
        dict(name="quantize_64k", op="quantize", B=1, Hkv=8, D=128, rows=65536, keep=0, dtype="bf16"),
        # an fp32 model's chosen rows, a head dimension that ends inside a group
        dict(name="quantize_chosen", op="quantize", B=2, Hkv=5, D=80, rows=2087, keep=1031, dtype="fp32"),
        # one sequence over its budget by a few rows, as in a chat: latency
        dict(name="evict_chat", op="evict", B=1, Hkv=8, D=128, rows=2111, spread=0.0, budget=2048, sinks=4, recent=64),
        # a serving batch of ragged caches, some below the budget
        dict(name="evict_batch", op="evict", B=16, Hkv=8, D=128, rows=9000, spread=0.7, budget=4096, sinks=4, recent=256),
        # a long document's cache cut to a quarter
        dict(name="evict_128k", op="evict", B=1, Hkv=8, D=128, rows=131072, spread=0.0, budget=32768, sinks=16,
             recent=1024),
        # a short chat: latency
        dict(name="attend_chat", op="attend", B=1, Hkv=8, G=4, D=128, rows=600, spread=0.0, ring=64, mass=False,
             dtype="bf16"),
        # one token after the 32K prompt at one key in four
        dict(name="attend_32k", op="attend", B=1, Hkv=8, G=4, D=128, rows=8297, spread=0.0, ring=128, mass=False,
             dtype="bf16"),
        # a serving batch of ragged fp16 caches that evict by weight
        dict(name="attend_batch", op="attend", B=16, Hkv=8, G=4, D=128, rows=9000, spread=0.7, ring=128, mass=True,
             dtype="fp16"),
        # four long documents
        dict(name="attend_4x128k", op="attend", B=4, Hkv=8, G=4, D=128, rows=131072, spread=0.0, ring=128, mass=True,
             dtype="bf16"),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["mass", "quantize", "evict", "attend"])
    D = rng.choice([40, 64, 80, 96, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    B, Hkv, G = rng.choice([1, 1, 2, 3, 8]), rng.choice([1, 2, 5, 8]), rng.choice([1, 2, 4, 4, 7, 8, 16])
    if op == "mass":
        anchors = rng.random() < 0.5
        Nk = _log(rng, 1, 32768)
        Nq = _log(rng, 1, 4096 if anchors else min(4096, Nk))
        while B * Hkv * G * Nq * Nk > 32 * 8192 * 4096:
            Nq = max(1, Nq // 2)
        return dict(op=op, B=B, Hkv=Hkv, G=G, D=D, Nq=Nq, Nk=Nk, anchors=anchors, dtype=dtype)
    rows = _log(rng, 1, 131072)
    if op == "quantize":
        rows = max(1, min(rows, 8 * 65536 // (B * Hkv)))
        return dict(op=op, B=B, Hkv=Hkv, D=D, rows=rows, keep=0 if rng.random() < 0.5 else _log(rng, 1, rows), dtype=dtype)
    spread = rng.choice([0.0, 0.3, 0.7])
    if op == "evict":
        rows = max(1, min(rows, 8 * 131072 // (B * Hkv)))
        budget = _log(rng, max(1, rows // 16), rows + 8)
        sinks = min(rng.choice([0, 4, 16]), budget)
        return dict(op=op, B=B, Hkv=Hkv, D=D, rows=rows, spread=spread, budget=budget, sinks=sinks,
                    recent=min(rng.choice([0, 1, 64, 256]), budget - sinks))
    rows = max(1, min(rows, 4 * 8 * 131072 // (B * Hkv * max(1, G // 4))))
    return dict(op=op, B=B, Hkv=Hkv, G=G, D=D, rows=rows, spread=spread, ring=rng.choice([1, 16, 50, 64, 128]),
                mass=rng.random() < 0.5, dtype=dtype)


def _lengths(case):
    """Rows of every (sequence, KV head): sequences shorten by up to ``spread`` along the batch,
    the heads of one differ by a few rows; at least one row."""
    B, H, rows = case["B"], case["Hkv"], case.get("rows", case.get("Nk"))
    per = [[max(1, int(rows * (1.0 - case.get("spread", 0.0) * b / B)) - (13 * h) % 29 * (rows > 64)) for h in range(H)]
           for b in range(B)]
    per[0][0] = rows
    return per


def _draw_rows(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _keys(gen, B, H, N, D, dtype):
    """Rows as projections give them, [B, N, H, D] seen as [B, H, N, D], with a few channels of
    larger size, as keys have them."""
    channel = torch.exp(0.5 * torch.randn(1, 1, H, D, generator=gen, device="cuda"))
    return (torch.randn(B, N, H, D, generator=gen, device="cuda") * channel).to(dtype).transpose(1, 2)


def _anchors(gen, B, H, N):
    """Run lengths 1 to 7 and the positions where the runs begin."""
    counts = torch.randint(1, 8, (B, H, N), generator=gen, device="cuda", dtype=torch.int32)
    return counts, (counts.cumsum(-1) - counts).to(torch.int32)


def _exponents(x):
    """Per group of 32 dims: the exponent of the smallest power of two with |x| <= 6 * 2^e."""
    _, e = torch.frexp(x)
    m = torch.ldexp(x, 3 - e)  # in [4, 8)
    return torch.where(m <= 6.0, e - 3, e - 2).clamp(-125, 125)


def _encode(rows):
    """Rows [..., D] -> codes [..., 16 * groups] and exponent bytes [..., groups], uint8."""
    D = rows.shape[-1]
    groups = (D + 31) // 32
    x = rows.float()
    if groups * 32 != D:
        x = torch.cat([x, x.new_zeros(*x.shape[:-1], groups * 32 - D)], -1)
    x = x.view(*x.shape[:-1], groups, 32)
    e = _exponents(x.abs().amax(-1))
    y = torch.ldexp(x.abs(), -e.unsqueeze(-1))
    # steps of 0.5 below 2, of 1 below 4, of 2 up to 6: round() takes ties to even
    code = torch.where(y < 2.0, torch.round(y * 2.0), torch.where(y < 4.0, torch.round(y) + 2.0, torch.round(y * 0.5) + 4.0))
    code = code.clamp(max=7.0).to(torch.uint8) | (torch.signbit(x).to(torch.uint8) << 3)
    code = code.view(*rows.shape[:-1], groups * 16, 2)
    return code[..., 0] | (code[..., 1] << 4), (e + 127).to(torch.uint8)


def _decode(codes, scales, D, dtype=torch.float32):
    """Codes and exponent bytes -> rows [..., D]."""
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device, dtype=dtype)
    x = level[torch.stack([codes & 15, codes >> 4], -1).view(*codes.shape[:-1], -1).int()]
    x = x.view(*scales.shape, 32) * torch.ldexp(torch.ones_like(scales, dtype=dtype), scales.int() - 127).unsqueeze(-1)
    return x.reshape(*codes.shape[:-1], -1)[..., :D]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op, B, H, D = case["op"], case["B"], case["Hkv"], case["D"]
    dtype = DTYPES[case.get("dtype", "bf16")]
    s = dict(case)
    if op == "mass":
        N, Nq, Hq = case["Nk"], case["Nq"], H * case["G"]
        s["q"] = _draw_rows(gen, B, Nq, Hq, D, dtype=dtype).transpose(1, 2)
        s["k"] = _keys(gen, B, H, N, D, dtype)
        s["counts"] = s["timestamps"] = s["lengths"] = None
        s["start"] = N - Nq
        if case["anchors"]:
            s["counts"], s["timestamps"] = _anchors(gen, B, H, N)
            s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
            s["start"] = 2 * N  # of about 4 N positions: later anchors are hidden from the queries
        return s
    N = case["rows"]
    s["counts"], s["timestamps"] = _anchors(gen, B, H, N)
    if op == "quantize":
        s["k"], s["v"] = _keys(gen, B, H, N, D, dtype), _draw_rows(gen, B, N, H, D, dtype=dtype).transpose(1, 2)
        s["index"] = None
        if case["keep"]:
            pick = torch.rand(B, H, N, generator=gen, device="cuda").argsort(-1)[..., :case["keep"]]
            s["index"] = pick.sort(-1).values.to(torch.int32)
        return s
    s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    s["k_codes"], s["k_scales"] = _encode(_keys(gen, B, H, N, D, torch.float32).contiguous())
    s["v_codes"], s["v_scales"] = _encode(_draw_rows(gen, B, H, N, D))
    # accumulated weights: a few heavy rows, a long tail, exact ties among the rows without any
    mass = torch.exp(3.0 * torch.randn(B, H, N, generator=gen, device="cuda") - 6.0)
    s["mass_sum"] = torch.where(mass < 1e-4, torch.zeros_like(mass), mass)
    if op == "attend":
        s["q"] = _draw_rows(gen, B, H * case["G"], 1, D, dtype=dtype)
        s["k_exact"], s["v_exact"] = (_draw_rows(gen, B, H, case["ring"], D, dtype=dtype) for _ in range(2))
    return s


# ---- plain forms -------------------------------------------------------------------------


def _softmax(scores):
    """Softmax over the last dim in place; a row of -inf gives zeros."""
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = scores.sum(-1, keepdim=True)
    return scores.div_(torch.where(total > 0, total, torch.ones_like(total)))


def _plain_mass(s):
    B, Hq, Nq, D = s["q"].shape
    H, N = s["k"].shape[1], s["k"].shape[2]
    q = s["q"].float().reshape(B, H, -1, D)
    p = torch.matmul(q, s["k"].float().transpose(-1, -2).contiguous()).mul_(D ** -0.5)
    row = torch.arange(N, device=p.device, dtype=torch.int32)
    seen = row.expand(B, H, N) if s["timestamps"] is None else s["timestamps"]
    p = p.view(B, H, Hq // H, Nq, N)
    if s["counts"] is not None:
        p.add_(s["counts"].float().log()[:, :, None, None])
    at = s["start"] + torch.arange(Nq, device=p.device)
    p.masked_fill_(seen[:, :, None, None] > at[:, None], -math.inf)
    if s["lengths"] is not None:
        p.masked_fill_((row >= s["lengths"][..., None])[:, :, None, None], -math.inf)
    return _softmax(p).sum((2, 3))


def _plain_quantize(s):
    k, v, counts, stamps = s["k"], s["v"], s["counts"], s["timestamps"]
    if s["index"] is not None:
        at = s["index"].long()
        k, v = (torch.gather(x, 2, at[..., None].expand(*at.shape, s["D"])) for x in (k, v))
        counts, stamps = torch.gather(counts, 2, at), torch.gather(stamps, 2, at)
    k, v = (_decode(*_encode(x), s["D"]).to(x.dtype) for x in (k, v))
    return {"k": k, "v": v, "counts": counts, "timestamps": stamps}


def _plain_evict(s):
    n, budget = s["lengths"].long(), s["budget"]
    N = s["mass_sum"].shape[-1]
    row = torch.arange(N, device=n.device).expand_as(s["mass_sum"])
    real = row < n[..., None]
    safe = real & ((row < s["sinks"]) | (row >= n[..., None] - s["recent"]))
    rank = torch.where(safe, math.inf, torch.where(real, s["mass_sum"], -math.inf))
    # most weight first, ties to the lowest row; rows past the length come last
    at = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    if at.shape[-1] < budget:
        at = torch.cat([at, at.new_full((*at.shape[:-1], budget - N), N)], -1)
    kept = n.clamp(max=budget)
    at = torch.where(torch.arange(budget, device=at.device) < kept[..., None], at, N).sort(-1).values
    gone, at = at >= N, at.clamp(max=N - 1)
    out = {"lengths": kept.to(torch.int32)}
    for name in ("counts", "timestamps", "mass_sum"):
        out[name] = torch.gather(s[name], 2, at).masked_fill_(gone, 0)
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
        x = s[name]
        out[name] = torch.gather(x, 2, at[..., None].expand(*at.shape, x.shape[-1])).masked_fill_(gone[..., None], 0)
    return out


def _plain_attend(s):
    B, Hq, _, D = s["q"].shape
    H, N, W = s["k_codes"].shape[1], s["k_codes"].shape[2], s["ring"]
    q = s["q"].float().view(B, H, Hq // H, D).transpose(-1, -2).contiguous()
    p = torch.cat([torch.matmul(_decode(s["k_codes"], s["k_scales"], D), q), torch.matmul(s["k_exact"].float(), q)], 2)
    p.mul_(D ** -0.5)
    p[:, :, :N].add_(s["counts"].float().log()[..., None])
    row = torch.arange(N, device=p.device, dtype=torch.int32)
    p[:, :, :N].masked_fill_((row >= s["lengths"][..., None])[..., None], -math.inf)
    p = _softmax(p.transpose(-1, -2).contiguous())
    out = torch.matmul(p[..., :N].contiguous(), _decode(s["v_codes"], s["v_scales"], D))
    out += torch.matmul(p[..., N:].contiguous(), s["v_exact"].float())
    out = out.view(B, Hq, 1, D).to(s["q"].dtype)
    return {"out": out, "mass_sum": s["mass_sum"] + p[..., :N].sum(2)} if s["mass"] else {"out": out}


_PLAIN = {"mass": _plain_mass, "quantize": _plain_quantize, "evict": _plain_evict, "attend": _plain_attend}


# ---- the framework's operators -----------------------------------------------------------


def _cache(ops, s, mass=None):
    return ops.KV4(k_codes=s["k_codes"], k_scales=s["k_scales"], v_codes=s["v_codes"], v_scales=s["v_scales"],
                   counts=s["counts"], timestamps=s["timestamps"], lengths=s["lengths"], head_dim=s["D"], mass=mass)


def _own(s):
    from deltaattention_amd import ops
    op = s["op"]
    if op == "mass":
        return ops.attention_mass(s["q"], s["k"], counts=s["counts"], timestamps=s["timestamps"], lengths=s["lengths"],
                                  q_start=s["start"])
    if op == "quantize":
        kv = ops.quantize_kv4(s["k"], s["v"], s["counts"], s["timestamps"], index=s["index"])
        k, v = ops.dequantize_kv4(kv, s["k"].dtype)
        return {"k": k, "v": v, "counts": kv.counts, "timestamps": kv.timestamps}
    if op == "evict":  # the rows' bytes are moved, not computed: they come as they are
        kv = ops.evict_kv4(_cache(ops, s, s["mass_sum"]), s["budget"], sinks=s["sinks"], recent=s["recent"])
        return {"lengths": kv.lengths, "counts": kv.counts, "timestamps": kv.timestamps, "mass_sum": kv.mass,
                "k_codes": kv.k_codes, "k_scales": kv.k_scales, "v_codes": kv.v_codes, "v_scales": kv.v_scales}
    # the call adds to the accumulated weights in place: a pass works on a copy of them
    mass = s["mass_sum"].clone() if s["mass"] else None
    out = ops.decode_attention_kv4(s["q"], _cache(ops, s, mass), s["k_exact"], s["v_exact"], s["ring"],
                                   accumulate=s["mass"])
    return {"out": out, "mass_sum": mass} if s["mass"] else {"out": out}


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------


def work(case):
    op, B, H, D = case["op"], case["B"], case["Hkv"], case["D"]
    es = ELEMENT.get(case.get("dtype"), 0)
    groups = (D + 31) // 32
    row4 = 2 * 17 * groups  # codes and exponents of a key and a value row
    if op == "mass":
        Nq, Nk, Hq = case["Nq"], case["Nk"], H * case["G"]
        start = 2 * Nk if case["anchors"] else Nk - Nq
        # keys that a query sees: all before it (anchors begin every 4 positions on average)
        seen = sum(min(Nk, (start + i) // 4 + 1) if case["anchors"] else start + i + 1 for i in range(Nq))
        return {"bytes": B * (Hq * Nq * D * es + H * Nk * D * es + H * Nk * (4 + 8 * case["anchors"])),
                "flops": 2.0 * B * Hq * D * seen}
    if op == "quantize":
        n = case["keep"] or case["rows"]
        return {"bytes": B * H * n * (2 * 2 * D * es + 16 + 4 * (case["keep"] > 0)), "flops": 4.0 * B * H * n * D}
    lengths = [n for per in _lengths(case) for n in per]
    if op == "evict":
        kept = sum(min(n, case["budget"]) for n in lengths)
        return {"bytes": sum(lengths) * 4 + kept * (row4 + 8) + B * H * case["budget"] * (row4 + 12),
                "flops": float(sum(lengths))}
    rows, G = sum(lengths), case["G"]
    return {"bytes": rows * (row4 + 4 + 8 * case["mass"]) + B * H * (2 * case["ring"] + 2 * G) * D * es,
            "flops": 4.0 * (rows + B * H * case["ring"]) * G * D}


# ---- the definitions in 64 bits --------------------------------------------------------------


def _exact_values(codes, scales, D):
    """Values of 4-bit rows from the bits of each element."""
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1).to(torch.int64)
    exponent, mantissa = (c >> 1) & 3, (c & 1).double()
    size = torch.where(exponent == 0, mantissa * 0.5, (1.0 + 0.5 * mantissa) * 2.0 ** (exponent - 1).double())
    power = torch.pow(2.0, scales.double() - 127.0).repeat_interleave(32, -1)
    return (torch.where(c >= 8, -size, size) * power)[..., :D]


def exact(case, seed):
    s = prepare(case, seed)
    op, B, H, D = case["op"], case["B"], case["Hkv"], case["D"]
    if op == "evict":  # whole numbers and rows moved as they are
        return None
    if op == "mass":
        out = torch.zeros(B, H, case["Nk"], dtype=torch.float64, device="cuda")
        place = torch.arange(case["Nk"], device="cuda")
        for b in range(B):
            for h in range(H):
                n = case["Nk"] if s["lengths"] is None else int(s["lengths"][b, h])
                keys = s["k"][b, h, :n].double().T.contiguous()
                stamp = place[:n] if s["timestamps"] is None else s["timestamps"][b, h, :n]
                size = 1.0 if s["counts"] is None else s["counts"][b, h, :n].double()
                for g in range(case["G"]):
                    for first in range(0, case["Nq"], 1024):
                        q = s["q"][b, h * case["G"] + g, first:first + 1024].double()
                        when = s["start"] + first + torch.arange(q.shape[0], device="cuda")
                        w = (q @ keys) / math.sqrt(D)
                        visible = stamp[None] <= when[:, None]
                        w = torch.exp(w - w.amax(-1, keepdim=True)) * size * visible
                        out[b, h, :n] += (w / w.sum(-1, keepdim=True).clamp(min=1e-300)).sum(0)
        return out
    if op == "quantize":
        got = {"counts": None, "timestamps": None}
        grid = torch.tensor(LEVELS, dtype=torch.float64, device="cuda")
        for name in ("k", "v"):
            x = s[name] if s["index"] is None else torch.take_along_dim(s[name], s["index"].long()[..., None], 2)
            x = torch.nn.functional.pad(x.double(), (0, -D % 32)).unflatten(-1, (-1, 32))
            top = x.abs().amax(-1, keepdim=True)
            power = torch.pow(2.0, torch.ceil(torch.log2(top / 6.0)).clamp(-125, 125))
            power = torch.where(power * 3.0 >= top, power * 0.5, power)  # log2 may be a step high at a border
            power = torch.where(power * 6.0 < top, power * 2.0, power)
            y = x.abs() / power
            above = torch.bucketize(y, grid).clamp(max=7)  # grid[above - 1] < y <= grid[above]
            below = (above - 1).clamp(min=0)
            up, down = grid[above] - y, y - grid[below]
            level = torch.where((up < down) | ((up == down) & (above % 2 == 0)), grid[above], grid[below])
            got[name] = (torch.copysign(level, x) * power).flatten(-2)[..., :D]
        return got
    G, W = case["G"], case["ring"]
    out = torch.zeros(B, H * G, 1, D, dtype=torch.float64, device="cuda")
    total = s["mass_sum"].double()
    for b in range(B):
        for h in range(H):
            n = int(s["lengths"][b, h])
            k, v = (torch.cat([_exact_values(s[x + "_codes"][b, h, :n], s[x + "_scales"][b, h, :n], D),
                               s[x + "_exact"][b, h].double()]) for x in "kv")
            size = torch.cat([s["counts"][b, h, :n].double(), torch.ones(W, dtype=torch.float64, device="cuda")])
            w = (s["q"][b, h * G:(h + 1) * G, 0].double() @ k.T.contiguous()) / math.sqrt(D)
            w = torch.exp(w - w.amax(-1, keepdim=True)) * size
            w = w / w.sum(-1, keepdim=True)
            out[b, h * G:(h + 1) * G, 0] = w @ v
            total[b, h, :n] += w[:, :n].sum(0)
    return {"out": out, "mass_sum": total} if case["mass"] else {"out": out}
