"""Cases of the three operators of a paged key/value cache at full width: writing new tokens into
it, attention of new tokens over it, and attention of a batch whose sequences share a prefix.

A case is a dict of plain values.  Its ``op`` names the operator:

* ``append``  ``ops.append_paged``: the keys of new tokens rotated to their positions and written,
  with their values, into the pages of their sequences; the queries rotated on the way;
* ``attend``  ``ops.paged_attention``: the new tokens of a ragged batch (one each in decoding, many
  in a prompt or a part of one) over the keys of their own sequence up to themselves;
* ``shared``  ``ops.shared_prefix_attention``: the same, where groups of sequences have the first
  tokens in common, whose pages are there once for the group.

Pages are [pages, Hkv, page size, D]; ``table`` [B, width] names each sequence's pages in order.
``lengths`` counts a sequence's tokens in its pages, the new ones included, so new token i of n is in
slot lengths - n + i.  Rotation is that of rotary position embeddings: the first ``rot`` dims in
pairs, (d, d + rot / 2) or with ``interleaved`` (2 d, 2 d + 1), by cos and sin of the position.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ELEMENT = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    llama = dict(Hq=32, Hkv=8, D=128, page=16, dtype="bf16")
    return [
        # a decode step of 64 sequences: latency
        dict(name="append_step", op="append", **llama, B=64, new=1, spread=0.0, past=450, rot=128, interleaved=False,
             per_token=False, start=0),
        # the whole 32K prompt of one sequence
        dict(name="append_prompt_32k", op="append", **llama, B=1, new=32768, spread=0.0, past=0, rot=128, interleaved=False,
             per_token=False, start=0),
        # ragged parts of prompts far into their sequences, partial rotation of neighbouring dims, odd heads
        dict(name="append_far", op="append", Hq=14, Hkv=2, D=96, page=64, dtype="fp16", B=7, new=411, spread=0.9, past=333,
             rot=64, interleaved=True, per_token=True, start=1000000),
        # one token of a short chat: latency
        dict(name="decode_chat", op="attend", **llama, B=1, new=1, spread=0.0, past=600),
        # a decode step of a ragged serving batch
        dict(name="decode_batch", op="attend", **llama, B=64, new=1, spread=0.8, past=9000),
        # one token after each of four long documents
        dict(name="decode_4x128k", op="attend", **llama, B=4, new=1, spread=0.0, past=131071),
        # the next part of a long prompt
        dict(name="prompt_part", op="attend", **llama, B=1, new=2048, spread=0.0, past=30011),
        # ragged whole prompts in fp16, heads in sevens
        dict(name="prompts", op="attend", Hq=28, Hkv=4, D=128, page=16, dtype="fp16", B=6, new=3001, spread=0.7, past=0),
        # a serving step: sequences that decode beside a part of a prompt
        dict(name="mixed_step", op="attend", **llama, B=16, new=512, spread=-1.0, past=5000),
        # the small fp32 layer (8 heads of 64 dims), a few tokens after a short chat
        dict(name="fp32_part", op="attend", Hq=8, Hkv=8, D=64, page=32, dtype="fp32", B=2, new=300, spread=0.3, past=211),
        # 16 answers sampled to one 32K prompt
        dict(name="shared_samples", op="shared", **llama, B=16, groups=1, prefix=32768, past=300, spread=0.5),
        # 128 chats over two long system prompts
        dict(name="shared_chats", op="shared", **llama, B=128, groups=2, prefix=8190, past=1000, spread=0.8),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "shared"])
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (8, 8), (8, 2), (6, 3), (28, 4), (16, 1)])
    c = dict(op=op, Hq=Hq, Hkv=Hkv, D=rng.choice([128, 128, 64, 80, 96]), page=rng.choice([16, 16, 32, 64, 256]),
             dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if op == "append":
        c.update(B=_log(rng, 1, 64), spread=rng.choice([0.0, 0.5, 0.9]), past=_log(rng, 1, 500),
                 rot=rng.choice([c["D"], c["D"], c["D"] // 2]), interleaved=rng.random() < 0.3, per_token=rng.random() < 0.3,
                 start=rng.choice([0, 0, 5000]))
        c["new"] = 1 if rng.random() < 0.3 else _log(rng, 2, 32768 // c["B"])
        return c
    if op == "shared":
        c.update(B=_log(rng, 2, 128), prefix=_log(rng, 64, 32768), past=_log(rng, 1, 1000), spread=rng.choice([0.0, 0.5, 0.8]))
        c["groups"] = min(c["B"], rng.choice([1, 1, 2, 3]))
        while c["B"] * (c["prefix"] + c["past"]) > 128 * 9000:
            c["prefix"] = (c["prefix"] + 1) // 2
        return c
    c.update(spread=rng.choice([0.0, 0.5, 0.8, -1.0]), B=_log(rng, 1, 64), past=_log(rng, 1, 131071))
    while c["B"] * c["past"] > 4 * 131072:
        c["past"] = (c["past"] + 1) // 2
    c["new"] = 1 if rng.random() < 0.5 else _log(rng, 2, 3000)
    while c["new"] > 1 and c["B"] * Hq * c["new"] * (c["past"] + c["new"]) > 32 * 2048 * (32000 if c["dtype"] != "fp32" else 8000):
        c["new"] = (c["new"] + 1) // 2
    return c


def _tokens(case):
    """(new tokens, tokens before them) of every sequence.  With ``spread`` -1 the first sequence
    brings ``new`` tokens and the others one; else both shorten by up to ``spread`` along the batch."""
    B, new, past = case["B"], case.get("new", 1), case["past"]
    if case["spread"] < 0:
        return [(new if b == 0 else 1, max(0, past - past * b // (2 * B) - 3 * b)) for b in range(B)]
    part = [1.0 - case["spread"] * b / B for b in range(B)]
    return [(max(1, int(new * p)), max(0, int(past * p) - b % 7 * (b > 0))) for b, p in enumerate(part)]


def _groups(case):
    """(first sequence, prefix tokens) of every group; a later group's prefix is a little shorter."""
    B, G = case["B"], case["groups"]
    return [(B * g // G, max(1, case["prefix"] - 37 * g)) for g in range(G)]


def _tables(gen, counts, page, more=3):
    """Pages of every sequence, taken in random order from a pool with a few to spare; -1 past them."""
    need = [-(-n // page) for n in counts]
    order = torch.randperm(sum(need) + more, generator=gen, device="cuda").to(torch.int32)
    width = max(max(need), 1)
    table = torch.full((len(need), width), -1, dtype=torch.int32, device="cuda")
    filled = torch.arange(width, device="cuda") < torch.tensor(need, device="cuda")[:, None]
    table[filled] = order[:sum(need)]
    return table, sum(need) + more


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s, dtype = dict(case), DTYPES[case["dtype"]]
    B, Hq, Hkv, D, page = case["B"], case["Hq"], case["Hkv"], case["D"], case["page"]
    tokens = _tokens(case)
    counts = [n + p for n, p in tokens]
    first = [sum(n for n, _ in tokens[:b]) for b in range(B + 1)]
    T = first[-1]
    s["max_new"] = max(n for n, _ in tokens)
    s["lengths"], s["cu"] = _ints(counts), _ints(first)
    prefix = _groups(case) if case["op"] == "shared" else []
    tables, pages = _tables(gen, counts + [n for _, n in prefix], page)
    s["table"] = tables[:B, :max(-(-n // page) for n in counts)].contiguous()
    if prefix:
        s["prefix_table"] = tables[B:].contiguous()
        s["prefix_lengths"] = _ints([n for _, n in prefix])
        s["prefix_cu"] = _ints([first[b] for b, _ in prefix] + [T])
        s["prefix_max"] = max(y - x for x, y in zip([b for b, _ in prefix], [b for b, _ in prefix[1:]] + [B]))
    # keys with a few channels of larger size, as keys have them
    channel = torch.exp(0.5 * torch.randn(1, Hkv, 1, D, generator=gen, device="cuda"))
    s["k_pages"] = (torch.randn(pages, Hkv, page, D, generator=gen, device="cuda") * channel).to(dtype)
    s["v_pages"] = torch.randn(pages, Hkv, page, D, generator=gen, device="cuda").to(dtype)
    if case["op"] != "append":
        s["q"] = torch.randn(T, Hq, D, generator=gen, device="cuda").to(dtype)
        return s
    # one projection's output, cut into queries, keys and values
    rows = torch.randn(T, Hq + 2 * Hkv, D, generator=gen, device="cuda").to(dtype)
    s["q"], s["k"], s["v"] = rows.split([Hq, Hkv, Hkv], 1)
    s["start"] = _ints([case["start"]] * B) if case["start"] else None
    at = torch.cat([torch.arange(p, p + n, device="cuda") for n, p in tokens]) if case["per_token"] else \
        torch.arange(max(counts), device="cuda")
    if case["per_token"]:
        at = at + case["start"]
    elif case["start"]:
        at = torch.arange(max(counts) + case["start"], device="cuda")
    half = case["rot"] // 2
    angle = at.double()[:, None] * torch.pow(500000.0, -torch.arange(half, device="cuda").double() / half)
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    return s


# ---- plain forms -------------------------------------------------------------------------


def _sequence_of(s):
    """The sequence of every token and the token's slot in its pages."""
    t = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.bucketize(t, s["cu"][1:].long(), right=True)
    return t, b, (s["lengths"][b] - s["cu"][b + 1] + t).long()


def _rotated(x, cos, sin, interleaved):
    half = cos.shape[-1]
    x = x.float()
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    cos, sin = cos[:, None], sin[:, None]
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _plain_append(s):
    t, b, slot = _sequence_of(s)
    at = t if s["per_token"] else slot if s["start"] is None else slot + s["start"][b]
    cos, sin = s["cos"][at], s["sin"][at]
    page = s["table"][b, slot // s["page"]].long()
    dtype = s["k"].dtype
    s["k_pages"][page, :, slot % s["page"]] = _rotated(s["k"], cos, sin, s["interleaved"]).to(dtype)
    s["v_pages"][page, :, slot % s["page"]] = s["v"]
    return {"q": _rotated(s["q"], cos, sin, s["interleaved"]).to(dtype), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _rows(pages, table):
    """[B, width] of pages -> [B, Hkv, width * page, D] in 32 bits."""
    x = pages[table.long().clamp(min=0)].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1]).float()


def _plain_attention(s, keys, values, seen):
    """Tokens padded to [B, most new tokens]; ``seen`` [B, new, keys]."""
    T, Hq, D = s["q"].shape
    t, b, _ = _sequence_of(s)
    B, H, N = keys.shape[:3]
    q = torch.zeros(B, s["max_new"], Hq, D, device="cuda")
    within = t - s["cu"][b]
    q[b, within] = s["q"].float()
    q = q.view(B, s["max_new"], H, Hq // H, D).permute(0, 2, 3, 1, 4).reshape(B, H, -1, D)
    p = torch.matmul(q, keys.transpose(-1, -2).contiguous()).mul_(D ** -0.5)
    p = p.view(B, H, Hq // H, s["max_new"], N).masked_fill_(~seen[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    out = torch.matmul(p.view(B, H, -1, N), values)
    out = out.view(B, H, Hq // H, s["max_new"], D).permute(0, 3, 1, 2, 4).reshape(B, s["max_new"], Hq, D)
    return out[b, within].to(s["q"].dtype)


def _before(s, N):
    """[B, new, N]: the slots up to each new token's own."""
    new = s["cu"][1:] - s["cu"][:-1]
    last = (s["lengths"] - new)[:, None] + torch.arange(s["max_new"], device="cuda")
    return torch.arange(N, device="cuda") <= last[..., None]


def _plain_attend(s):
    keys, values = _rows(s["k_pages"], s["table"]), _rows(s["v_pages"], s["table"])
    return {"out": _plain_attention(s, keys, values, _before(s, keys.shape[2]))}


def _plain_shared(s):
    group = torch.bucketize(s["cu"][:-1].long(), s["prefix_cu"][1:].long(), right=True)
    table = torch.cat([s["prefix_table"][group], s["table"]], 1)
    N = s["prefix_table"].shape[1] * s["page"]
    common = torch.arange(N, device="cuda") < s["prefix_lengths"][group][:, None]
    mine = _before(s, s["table"].shape[1] * s["page"])
    seen = torch.cat([common[:, None].expand(-1, s["max_new"], -1), mine], 2)
    return {"out": _plain_attention(s, _rows(s["k_pages"], table), _rows(s["v_pages"], table), seen)}


_PLAIN = {"append": _plain_append, "attend": _plain_attend, "shared": _plain_shared}


# ---- the framework's operators -----------------------------------------------------------


def _own(s):
    from deltaattention_amd import ops
    kv = ops.PagedKV(s["k_pages"], s["v_pages"])
    if s["op"] == "append":
        batch = ops.PagedBatch(s["table"], s["lengths"], s["cu"], s["max_new"], start=s["start"])
        q = ops.append_paged(kv, batch, s["k"], s["v"], q=s["q"], cos=s["cos"], sin=s["sin"],
                             interleaved=s["interleaved"], per_token=s["per_token"])
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    batch = ops.PagedBatch(s["table"], s["lengths"], s["cu"], s["max_new"])
    if s["op"] == "attend":
        return {"out": ops.paged_attention(s["q"], kv, batch)}
    prefix = ops.PagedBatch(s["prefix_table"], s["prefix_lengths"], s["prefix_cu"], s["prefix_max"])
    return {"out": ops.shared_prefix_attention(s["q"], kv, batch, prefix)}


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------


def work(case):
    Hq, Hkv, D, es, page = case["Hq"], case["Hkv"], case["D"], ELEMENT[case["dtype"]], case["page"]
    tokens = _tokens(case)
    T = sum(n for n, _ in tokens)
    if case["op"] == "append":
        table = T if case["per_token"] else len(set().union(*(range(p, p + n) for n, p in tokens)))
        return {"bytes": 2 * T * (Hq + 2 * Hkv) * D * es + table * case["rot"] * 4 + 4 * T // page,
                "flops": 3.0 * T * (Hq + Hkv) * case["rot"]}
    keys = sum(n + p for n, p in tokens)
    seen = sum(n * p + n * (n + 1) // 2 for n, p in tokens)
    if case["op"] == "shared":
        groups = _groups(case) + [(case["B"], 0)]
        keys += sum(n for _, n in groups)
        seen += sum(n * (groups[g + 1][0] - b) for g, (b, n) in enumerate(groups[:-1]))
    return {"bytes": 2 * T * Hq * D * es + 2 * keys * Hkv * D * es + 4 * keys // page, "flops": 4.0 * D * Hq * seen}


# ---- the definitions in 64 bits --------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    D, page, G = case["D"], case["page"], case["Hq"] // case["Hkv"]
    tokens = _tokens(case)
    cu = s["cu"].tolist()
    if case["op"] == "append":
        half, pages = case["rot"] // 2, {x: s[x + "_pages"].double() for x in "kv"}
        turned = {}
        where = torch.cat([torch.arange(p, p + n, device="cuda") + case["start"] for n, p in tokens])
        row = torch.arange(len(where), device="cuda") if case["per_token"] else where
        wheel = torch.complex(s["cos"][row].double(), s["sin"][row].double())[:, None]
        for name in "qk":
            x = s[name].double().clone()
            d = torch.arange(half, device="cuda")
            one, two = (2 * d, 2 * d + 1) if case["interleaved"] else (d, d + half)
            z = torch.complex(x[..., one], x[..., two]) * wheel
            x[..., one], x[..., two] = z.real, z.imag
            turned[name] = x
        for b, (n, p) in enumerate(tokens):
            for i in range(n) if n <= 64 else ():
                at = int(s["table"][b, (p + i) // page])
                pages["k"][at, :, (p + i) % page] = turned["k"][cu[b] + i]
                pages["v"][at, :, (p + i) % page] = s["v"][cu[b] + i].double()
            if n > 64:
                slot = torch.arange(p, p + n, device="cuda")
                at = s["table"][b].long()[slot // page]
                pages["k"][at, :, slot % page] = turned["k"][cu[b]:cu[b + 1]]
                pages["v"][at, :, slot % page] = s["v"][cu[b]:cu[b + 1]].double()
        return {"q": turned["q"], "k_pages": pages["k"], "v_pages": pages["v"]}
    out = torch.zeros(cu[-1], case["Hq"], D, dtype=torch.float64, device="cuda")
    groups = _groups(case) if case["op"] == "shared" else []
    for b, (n, p) in enumerate(tokens):
        at, common = s["table"][b, :-(-(n + p) // page)].long(), 0
        pick = [(at, n + p)]
        if groups:
            g = max(i for i, (first, _) in enumerate(groups) if first <= b)
            common = groups[g][1]
            pick.insert(0, (s["prefix_table"][g, :-(-common // page)].long(), common))
        for h in range(case["Hkv"]):
            k, v = (torch.cat([s[x + "_pages"][i, h].reshape(-1, D)[:m].double() for i, m in pick]) for x in "kv")
            for first in range(0, n, 1024):
                q = s["q"][cu[b] + first:cu[b] + min(n, first + 1024), h * G:(h + 1) * G].double()
                when = common + p + first + torch.arange(q.shape[0], device="cuda")
                w = (q.reshape(-1, D) @ k.T.contiguous()).view(q.shape[0], G, -1) / math.sqrt(D)
                w = w.masked_fill((torch.arange(k.shape[0], device="cuda") > when[:, None])[:, None], -math.inf)
                w = torch.softmax(w, -1)
                out[cu[b] + first:cu[b] + first + q.shape[0], h * G:(h + 1) * G] = (w.view(-1, k.shape[0]) @ v).view_as(q)
    return {"out": out}
