"""The paged cache's operators against their 64-bit definitions."""
import pytest
import torch

import paged_reference as R
from conftest import announce

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _cu(new):
    return [sum(new[:b]) for b in range(len(new) + 1)]


class World:
    """Pages and sequences; ``new`` and ``past`` tokens of every sequence, ``prefix`` [(sequences, tokens)]."""

    def __init__(self, new, past, Hq, Hkv, D, page, dtype, prefix=(), seed=0, junk=True, scale_k=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.lengths = [n + p for n, p in zip(new, past)]
        self.cu = _cu(new)
        self.Hq, self.Hkv, self.D, self.page, self.dtype = Hq, Hkv, D, page, DT[dtype]
        counts = self.lengths + [n for _, n in prefix]
        table, P = R.tables(counts, page, gen=gen)
        B = len(new)
        self.table, self.prefix = table[:B].contiguous(), None
        self.k, self.v = (torch.randn(P, Hkv, page, D, generator=gen) for _ in range(2))
        self.k = (self.k * scale_k).to(self.dtype)
        self.v = self.v.to(self.dtype)
        if junk:  # what no sequence holds may be anything
            used = torch.zeros(P, page, dtype=torch.bool)
            for b, n in enumerate(counts):
                for j in range(-(-n // page)):
                    used[table[b, j], :min(page, n - j * page)] = True
            for pages, bad in ((self.k, float("nan")), (self.v, float("inf"))):
                pages.masked_fill_(~used[:, None, :, None], bad)
        self.q = torch.randn(self.cu[-1], Hq, D, generator=gen).to(self.dtype)
        if prefix:
            first = _cu([m for m, _ in prefix])
            self.prefix = (table[B:].contiguous(), [n for _, n in prefix], [self.cu[b] for b in first])

    def batch(self, ops, **more):
        return ops.PagedBatch(self.table.cuda(), _i(self.lengths), self.cu, **more)

    def call(self, ops, q=None, kv=None, batch=None, out=None, scale=None):
        kv = ops.PagedKV(self.k.cuda(), self.v.cuda()) if kv is None else kv
        q = self.q.cuda() if q is None else q
        batch = self.batch(ops) if batch is None else batch
        if self.prefix is None:
            return ops.paged_attention(q, kv, batch, scale=scale, out=out)
        t, n, cu = self.prefix
        return ops.shared_prefix_attention(q, kv, batch, ops.PagedBatch(t.cuda(), _i(n), cu), scale=scale, out=out)

    def want(self, scale=None):
        return R.attention(self.q, self.k, self.v, self.table, self.lengths, self.cu, self.prefix, scale)

    def check(self, got, scale=None):
        want, tol = self.want(scale)
        close(got, want, tol)


def _i(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def close(got, want, tol):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    off = (got - want).abs() - tol
    at = off.argmax()
    assert off.max() <= 0, f"off by {(got - want).abs().flatten()[at]:.3e}, allowed {tol.flatten()[at]:.3e} at {int(at)}"


HEADS = [(8, 2), (4, 4), (14, 2), (6, 3), (16, 1), (32, 8)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Hq,Hkv", HEADS)
def test_decode(gpu, Hq, Hkv, dtype):
    """One token each: lengths of one to a few tiles, page and tile borders among them."""
    from deltaattention_amd import ops
    announce(f"paged decode {Hq}/{Hkv} {dtype}")
    past = [0, 1, 14, 15, 16, 30, 31, 32, 63, 64, 126, 127, 128, 200, 511, 777]
    w = World([1] * len(past), past, Hq, Hkv, 128, 16, dtype)
    w.check(w.call(ops))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("Hq,Hkv", [(64, 1), (33, 1), (66, 2), (32, 1)])
def test_many_heads_to_one(gpu, Hq, Hkv, dtype):
    """Groups of 32 query heads and more: a token alone is more rows than the stream takes."""
    from deltaattention_amd import ops
    announce(f"paged attention {Hq}/{Hkv} {dtype}")
    w = World([1, 3, 0, 1], [700, 40, 9, 0], Hq, Hkv, 64, 16, dtype, prefix=[(2, 90), (2, 17)])
    w.check(w.call(ops))
    w.prefix = None
    w.check(w.call(ops))


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("B,long", [(300, 0), (700, 3), (257, 1)])
def test_many_sequences(gpu, B, long, wide):
    """More sequences than a workgroup has threads, some of them long or without tokens; a table with room
    for long ones (`wide`) has the keys of all go as one stream."""
    from deltaattention_amd import ops
    announce(f"paged attention of {B} sequences, {long} long, wide={wide}")
    new = [0 if b % 50 == 7 else 1 for b in range(B)]
    past = [(b * 7) % 60 + (3000 if b % 90 == 5 and b // 90 < long else 0) for b in range(B)]
    new[B // 2] = 45 if long else 1
    w = World(new, past, 8, 2, 64, 16, "bf16")
    if wide:
        w.table = torch.cat([w.table, torch.full((B, 300), -1, dtype=torch.int32)], 1)
    w.check(w.call(ops))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_more_tokens_than_max_seqlen(gpu, dtype):
    """A sequence with more tokens than max_seqlen is cut to it; the others are as they should be."""
    from deltaattention_amd import ops
    announce(f"paged attention, max_seqlen too small {dtype}")
    w = World([5, 300, 1, 40], [10, 20, 400, 7], 8, 2, 64, 16, dtype)
    got = ops.paged_attention(w.q.cuda(), ops.PagedKV(w.k.cuda(), w.v.cuda()),
                              ops.PagedBatch(w.table.cuda(), _i(w.lengths), _i(w.cu), 40)).double().cpu()
    want, tol = w.want()
    for a, b in ((0, 5), (305, 306), (306, 346)):
        assert ((got[a:b] - want[a:b]).abs() <= tol[a:b]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [8, 40, 64, 80, 96, 120])
def test_head_dims(gpu, D, dtype):
    from deltaattention_amd import ops
    announce(f"paged attention D={D} {dtype}")
    w = World([1, 3, 70, 1], [129, 20, 50, 0], 8, 2, D, 32, dtype)
    w.check(w.call(ops))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 512])
def test_page_sizes(gpu, page, dtype):
    from deltaattention_amd import ops
    announce(f"paged attention page={page} {dtype}")
    w = World([1, 100, 1, 5], [1000, 333, 0, 64], 8, 2, 64, page, dtype)
    w.check(w.call(ops))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Hq,Hkv", HEADS)
@pytest.mark.parametrize("n", [2, 9, 65, 200, 333])
def test_prompts(gpu, n, Hq, Hkv, dtype):
    """Whole prompts and parts of prompts of one ragged batch."""
    from deltaattention_amd import ops
    announce(f"paged prompts {n} {Hq}/{Hkv} {dtype}")
    w = World([n, 1, n // 2 + 1, 0, n], [0, 40, 77, 0, 129], Hq, Hkv, 128, 16, dtype)
    w.check(w.call(ops))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("past", [4000, 20011])
def test_long(gpu, past, dtype):
    """Long caches of few heads: keys split over the chip and joined."""
    from deltaattention_amd import ops
    announce(f"paged long {past} {dtype}")
    w = World([1, 1, 4], [past, 13, past // 3], 8, 2, 128, 16, dtype)
    w.check(w.call(ops))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_part_after_long(gpu, dtype):
    from deltaattention_amd import ops
    announce(f"paged part of a prompt after 6000 tokens {dtype}")
    w = World([67, 1, 130], [6000, 2500, 1111], 8, 2, 128, 16, dtype)
    w.check(w.call(ops))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Hq,Hkv", HEADS)
@pytest.mark.parametrize("prefix", [[(5, 700)], [(2, 33), (3, 1)], [(1, 300), (3, 0), (1, 129)]])
def test_shared_prefix(gpu, prefix, Hq, Hkv, dtype):
    from deltaattention_amd import ops
    announce(f"shared prefix {prefix} {Hq}/{Hkv} {dtype}")
    w = World([1] * 5, [0, 17, 130, 64, 5], Hq, Hkv, 128, 16, dtype, prefix=prefix)
    w.check(w.call(ops))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("B,prefix", [(40, 3000), (3, 9000), (130, 257)])
def test_shared_prefix_batches(gpu, B, prefix, dtype):
    from deltaattention_amd import ops
    announce(f"shared prefix of {B} sequences, {prefix} tokens {dtype}")
    w = World([1] * B, [(37 * b) % 150 for b in range(B)], 8, 2, 64, 32, dtype, prefix=[(B // 2, prefix), (B - B // 2, prefix // 3)])
    w.check(w.call(ops))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_shared_prefix_prompts(gpu, dtype):
    """Sequences behind a prefix that bring many tokens, or none."""
    from deltaattention_amd import ops
    announce(f"shared prefix, many tokens {dtype}")
    w = World([70, 1, 0, 9], [3, 100, 50, 0], 8, 2, 128, 16, dtype, prefix=[(3, 200), (1, 77)])
    w.check(w.call(ops))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_nothing_to_see(gpu, dtype):
    """Sequences that are shorter than what they bring: the first tokens see nothing and give zeros."""
    from deltaattention_amd import ops
    announce(f"paged attention without keys {dtype}")
    w = World([1, 5, 1, 40], [0, 0, 3, 0], 8, 2, 64, 16, dtype)
    w.lengths = [0, 2, 4, 0]
    got = w.call(ops)
    w.check(got)
    assert (got[0] == 0).all() and (got[1:4] == 0).all() and (got[7:] == 0).all() and (got[4:7] != 0).any()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_large_scores(gpu, dtype):
    """Scores of some hundreds: the running maximum moves, most weights vanish."""
    from deltaattention_amd import ops
    announce(f"paged attention, large scores {dtype}")
    w = World([1, 90, 1], [600, 10, 3], 8, 2, 128, 16, dtype, scale_k=30.0)
    w.check(w.call(ops))
    w.check(w.call(ops, scale=0.01), scale=0.01)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("new", [[1, 1, 1], [1, 40, 3]])
def test_strides(gpu, new, dtype):
    """Pages as [pages, page, heads, D], queries cut from a wider projection, an output with gaps, a
    table that is wider than the sequences and part of a larger one."""
    from deltaattention_amd import ops
    announce(f"paged strides {new} {dtype}")
    w = World(new, [50, 3, 200], 8, 2, 64, 16, dtype)
    k, v = (x.transpose(1, 2).contiguous().cuda().transpose(1, 2) for x in (w.k, w.v))
    T = w.cu[-1]
    wide = torch.zeros(T, 12, 64, dtype=w.dtype, device="cuda")
    wide[:, 2:10] = w.q.cuda()
    big = torch.full((T, 10, 72), 7.0, dtype=w.dtype, device="cuda")
    table = torch.full((4, 40), 1 << 30, dtype=torch.int32, device="cuda")
    table[:3, 2:2 + w.table.shape[1]] = w.table.cuda()
    batch = ops.PagedBatch(table[:3, 2:], _i(w.lengths), w.cu)
    out = big[:, 1:9, :64]
    got = w.call(ops, q=wide[:, 2:10], kv=ops.PagedKV(k, v), batch=batch, out=out)
    assert got is out
    w.check(out)
    assert (big[:, 0] == 7).all() and (big[:, 9] == 7).all() and (big[:, :, 64:] == 7).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("prefix", [(), [(2, 100), (2, 30)]])
def test_padded_batch(gpu, prefix, dtype):
    """Tokens past the last sequence keep what the output held; sequences without tokens among others."""
    from deltaattention_amd import ops
    announce(f"paged padded batch {dtype}")
    w = World([1, 0, 60, 2], [300, 10, 20, 0], 8, 2, 64, 16, dtype, prefix=prefix)
    T = w.cu[-1]
    q = torch.full((T + 9, 8, 64), float("nan"), dtype=w.dtype, device="cuda")
    q[:T] = w.q.cuda()
    out = torch.full_like(q, 3.0)
    w.call(ops, q=q, out=out)
    w.check(out[:T])
    assert (out[T:] == 3).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_same_results_again(gpu, dtype):
    """Two runs agree bit for bit, and a sequence's result is its own: other sequences do not change
    which keys it sees."""
    from deltaattention_amd import ops
    announce(f"paged attention twice {dtype}")
    w = World([1, 33, 1, 1], [5000, 200, 31, 2222], 8, 2, 128, 16, dtype)
    kv, batch, q = ops.PagedKV(w.k.cuda(), w.v.cuda()), w.batch(ops), w.q.cuda()
    one = w.call(ops, q, kv, batch)
    for _ in range(3):
        assert torch.equal(one, w.call(ops, q, kv, batch))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("new", [1, 5, 70])
def test_bad_pages_are_not_touched(gpu, new, dtype):
    """Entries that name no page, where a sequence needs them: zeros in their place."""
    from deltaattention_amd import ops
    announce(f"paged attention, entries outside the pool, {new} tokens {dtype}")
    w = World([new, new, new], [300, 40, 129], 8, 2, 64, 16, dtype)
    w.table[0, 3] = -1
    w.table[0, 7] = 1 << 30
    w.table[1, 0] = w.k.shape[0]
    w.table[2, 2] = -(1 << 31)
    w.check(w.call(ops))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_malformed_batches_stay_inside(gpu, dtype):
    """Lengths and cu_seqlens that contradict each other are clamped; no row outside is written."""
    from deltaattention_amd import ops
    announce(f"paged attention, malformed lengths {dtype}")
    w = World([1, 2, 40], [50, 3, 9], 8, 2, 64, 16, dtype, junk=False)
    T = w.cu[-1]
    kv, q = ops.PagedKV(w.k.cuda(), w.v.cuda()), w.q.cuda()
    for lengths, cu in (([1 << 30, -5, 1 << 30], w.cu), (w.lengths, [0, 1000, 20, T]), (w.lengths, [-7, 5, 3, 1 << 30])):
        whole = torch.full((T + 8, 8, 64), 3.0, dtype=w.dtype, device="cuda")
        batch = ops.PagedBatch(w.table.cuda(), _i(lengths), _i(cu), 40)
        ops.paged_attention(q, kv, batch, out=whole[4:T + 4])
        torch.cuda.synchronize()
        assert (whole[:4] == 3).all() and (whole[T + 4:] == 3).all()
        k0 = kv.k_pages.clone()
        x = torch.ones(T, 2, 64, dtype=w.dtype, device="cuda")
        ops.append_paged(kv, batch, x, x)
        torch.cuda.synchronize()
        kv.k_pages.copy_(k0)


def _rope(rows, rot, dtype=torch.float32, first=0):
    half = rot // 2
    angle = (torch.arange(rows).double() + first)[:, None] * 10000.0 ** (-torch.arange(half).double() / half)
    return angle.cos().to(dtype), angle.sin().to(dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (80, 80), (80, 40), (96, 36), (72, 20), (8, 8), (40, 4), (64, 0)])
def test_append(gpu, D, rot, interleaved, dtype):
    from deltaattention_amd import ops
    announce(f"append D={D} rot={rot} interleaved={interleaved} {dtype}")
    new, past = [1, 40, 0, 7, 16], [0, 13, 5, 100, 16]
    w = World(new, past, 14, 2, D, 16, dtype, junk=False, seed=3)
    T = w.cu[-1]
    gen = torch.Generator().manual_seed(9)
    proj = torch.randn(T, 18, D, generator=gen).to(w.dtype)
    q, k, v = proj.split([14, 2, 2], 1)
    dev = proj.cuda()
    dq, dk, dv = dev.split([14, 2, 2], 1)
    kv = ops.PagedKV(w.k.cuda(), w.v.cuda())
    at = torch.tensor([w.lengths[b] - new[b] + i for b in range(5) for i in range(new[b])])
    if rot:
        cos, sin = _rope(200, rot)
        turn = lambda x: R.rotate(x, cos[at], sin[at], interleaved)  # noqa: E731
        got = ops.append_paged(kv, w.batch(ops), dk, dv, q=dq, cos=cos.cuda(), sin=sin.cuda(), interleaved=interleaved)
    else:
        turn = lambda x: (x.double(), torch.zeros_like(x, dtype=torch.float64))  # noqa: E731
        got = ops.append_paged(kv, w.batch(ops), dk, dv, q=dq)
    close(got, *turn(q))
    want_k, want_v, tol = w.k.double(), w.v.double(), torch.zeros_like(w.k, dtype=torch.float64)
    turned, ktol = turn(k)
    for t in range(T):
        b = next(b for b in range(5) if w.cu[b] <= t < w.cu[b + 1])
        page, row = int(w.table[b, at[t] // 16]), int(at[t] % 16)
        want_k[page, :, row], tol[page, :, row], want_v[page, :, row] = turned[t], ktol[t], v[t].double()
    close(kv.k_pages, want_k, tol)
    assert torch.equal(kv.v_pages.double().cpu(), want_v)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_append_positions(gpu, dtype):
    """Rows by token, positions behind a prefix, cos and sin in the pages' type, without queries, in place."""
    from deltaattention_amd import ops
    announce(f"append positions {dtype}")
    w = World([3, 1, 20], [20, 0, 1], 4, 2, 64, 32, dtype, junk=False)
    T = w.cu[-1]
    gen = torch.Generator().manual_seed(2)
    k, v, q = (torch.randn(T, h, 64, generator=gen).to(w.dtype) for h in (2, 2, 4))
    start = [7, 100, 0]
    seq = [b for b in range(3) for _ in range(w.cu[b + 1] - w.cu[b])]
    slot = torch.tensor([w.lengths[b] - w.cu[b + 1] + t for t, b in enumerate(seq)])
    pos = slot + torch.tensor([start[b] for b in seq])
    cos, sin = _rope(300, 64)
    page = torch.stack([w.table[b, s // 32] for b, s in zip(seq, slot)]).long()

    def check(got_q, kv, c, s):
        if got_q is not None:
            close(got_q, *R.rotate(q, c, s, False))
        close(kv.k_pages[page.cuda(), :, (slot % 32).cuda()], *R.rotate(k, c, s, False))
    kv = ops.PagedKV(w.k.cuda(), w.v.cuda())
    batch = w.batch(ops, start=_i(start))
    dq = q.cuda()
    got = ops.append_paged(kv, batch, k.cuda(), v.cuda(), q=dq, cos=cos.cuda(), sin=sin.cuda(), out=dq)
    assert got is dq
    check(got, kv, cos[pos], sin[pos])
    kv = ops.PagedKV(w.k.cuda(), w.v.cuda())
    assert ops.append_paged(kv, batch, k.cuda(), v.cuda(), cos=cos.cuda(), sin=sin.cuda()) is None
    check(None, kv, cos[pos], sin[pos])
    low = (torch.cat([x, x], 1).to(w.dtype)[pos] for x in (cos, sin))  # a row each, both halves, as models make them
    c, s = (x.cuda()[:, :32] for x in low)
    kv = ops.PagedKV(w.k.cuda(), w.v.cuda())
    got = ops.append_paged(kv, w.batch(ops), k.cuda(), v.cuda(), q=q.cuda(), cos=c, sin=s, per_token=True)
    check(got, kv, c.cpu().float(), s.cpu().float())


def test_append_leaves_the_rest(gpu):
    """Tokens past the last sequence, places past the table, pages that are not there and sequences
    shorter than what they bring: nothing else is written."""
    from deltaattention_amd import ops
    announce("append: what is not written")
    w = World([2, 3, 1], [30, 15, 0], 4, 2, 64, 16, "bf16", junk=False)
    w.table[1, 1] = -1           # its tokens 16 and 17; token 15 stays
    kv = ops.PagedKV(w.k.cuda(), w.v.cuda())
    T = 6
    x = torch.ones(T + 3, 2, 64, dtype=torch.bfloat16, device="cuda")
    q = torch.randn(T + 3, 4, 64, device="cuda").to(torch.bfloat16)
    out = torch.full_like(q, 5.0)
    lengths = [32, 18, 0]        # the last sequence has no place for its token
    ops.append_paged(kv, ops.PagedBatch(w.table.cuda(), _i(lengths), w.cu), x, x, q=q, out=out)
    want = w.k.clone()
    for b, s in ((0, 30), (0, 31), (1, 15)):
        want[w.table[b, s // 16], :, s % 16] = 1
    assert torch.equal(kv.k_pages.cpu(), want)
    assert torch.equal(out[:T], q[:T]) and (out[T:] == 5).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("prefix", [(), [(4, 150)]])
def test_captured_steps(gpu, prefix, dtype):
    """A decode step (rotation, write, attention) captured once and replayed as the sequences grow,
    each replay against the eager calls, with eager work between."""
    from deltaattention_amd import ops
    announce(f"paged steps captured {dtype}")
    steps, B = 6, 4
    w = World([1] * B, [100, 15, 0, 31], 8, 2, 64, 16, dtype, prefix=prefix, junk=False)
    counts = [n + steps for n in w.lengths] + ([n for _, n in prefix])
    table, P = R.tables(counts, 16, gen=torch.Generator().manual_seed(4))
    ptable = table[B:].contiguous().cuda()
    table = table[:B].contiguous().cuda()
    gen = torch.Generator().manual_seed(5)
    base_k, base_v = (torch.randn(P, 2, 16, 64, generator=gen).to(w.dtype).cuda() for _ in range(2))
    data = [[torch.randn(B, h, 64, generator=gen).to(w.dtype).cuda() for h in (8, 2, 2)] for _ in range(steps)]
    cos, sin = (x.cuda() for x in _rope(400, 64))
    start = _i([150] * B) if prefix else None
    pre = ops.PagedBatch(ptable, _i([150]), _i([0, B]), B) if prefix else None

    def step(kv, batch, q, k, v):
        q = ops.append_paged(kv, batch, k, v, q=q, cos=cos, sin=sin)
        return ops.shared_prefix_attention(q, kv, batch, pre) if prefix else ops.paged_attention(q, kv, batch)
    eager, kv, lengths = [], ops.PagedKV(base_k.clone(), base_v.clone()), _i(w.lengths)
    for x in data:
        eager.append(step(kv, ops.PagedBatch(table, lengths, start=start), *x))
        lengths = lengths + 1
    kv, lengths = ops.PagedKV(base_k.clone(), base_v.clone()), _i(w.lengths)
    batch = ops.PagedBatch(table, lengths, start=start)
    still = [t.clone() for t in data[0]]
    step(kv, batch, *still)  # warm
    kv.k_pages.copy_(base_k)
    kv.v_pages.copy_(base_v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(kv, batch, *still)
    for i, x in enumerate(data):
        for a, b in zip(still, x):
            a.copy_(b)
        graph.replay()
        assert torch.equal(out, eager[i]), i
        other = World([1, 20], [40, 3], 8, 2, 64, 16, dtype)
        other.check(other.call(ops))
        torch.cuda.synchronize()
        lengths += 1


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("new,past,prefix", [([70, 1, 33], [5000, 900, 3], ()), ([1] * 40, [30] * 40, [(25, 2000), (15, 90)]),
                                             ([3] * 12, [10] * 12, [(12, 700)]), ([300], [0], ())])
def test_captured_attention(gpu, new, past, prefix, dtype):
    """Every kernel's launches captured and replayed on other queries, with eager calls between."""
    from deltaattention_amd import ops
    announce(f"paged attention captured {new[:3]} {prefix} {dtype}")
    w = World(new, past, 8, 2, 64, 16, dtype, prefix=prefix)
    kv, batch = ops.PagedKV(w.k.cuda(), w.v.cuda()), w.batch(ops)
    pre = None if not prefix else ops.PagedBatch(w.prefix[0].cuda(), _i(w.prefix[1]), w.prefix[2])

    def call(q):
        return ops.shared_prefix_attention(q, kv, batch, pre) if prefix else ops.paged_attention(q, kv, batch)
    gen = torch.Generator().manual_seed(8)
    qs = [torch.randn(w.q.shape, generator=gen).to(w.dtype).cuda() for _ in range(4)]
    eager = [call(q) for q in qs]
    still = qs[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(still)
    for q, want in zip(qs, eager):
        still.copy_(q)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(call(q), want)
    w.q = qs[-1].cpu()
    w.check(out)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("new", [1, 40])
def test_sequences_outside_every_group(gpu, new, dtype):
    """Tokens before the first group and after the last see their own sequence alone."""
    from deltaattention_amd import ops
    announce(f"shared prefix, sequences outside the groups, {new} tokens {dtype}")
    w = World([new] * 6, [3 * b for b in range(6)], 8, 2, 64, 16, dtype, prefix=[(2, 100), (3, 55), (1, 9)])
    t, n, cu = w.prefix
    w.prefix = (t[:2], n[:2], [2 * new, 4 * new, 5 * new])
    pre = ops.PagedBatch(w.prefix[0].cuda(), _i(w.prefix[1]), _i(w.prefix[2]), 2 * new)
    w.check(ops.shared_prefix_attention(w.q.cuda(), ops.PagedKV(w.k.cuda(), w.v.cuda()), w.batch(ops), pre))


def test_two_streams_at_once(gpu):
    """Calls of every kernel in flight on two streams: no memory is shared between calls."""
    from deltaattention_amd import ops
    announce("paged attention on two streams at once")
    worlds = [World([1] * 9, [4000 + 7 * b for b in range(9)], 8, 2, 64, 16, "bf16"),
              World([200, 1, 3], [900, 5000, 0], 8, 2, 64, 16, "bf16"),
              World([1] * 30, [20] * 30, 8, 2, 64, 16, "bf16", prefix=[(30, 3000)])]
    calls = []
    for w in worlds:
        kv, batch, q = ops.PagedKV(w.k.cuda(), w.v.cuda()), w.batch(ops), w.q.cuda()
        pre = None if w.prefix is None else ops.PagedBatch(w.prefix[0].cuda(), _i(w.prefix[1]), w.prefix[2])
        calls.append((lambda q=q, kv=kv, batch=batch: ops.paged_attention(q, kv, batch)) if pre is None else
                     (lambda q=q, kv=kv, batch=batch, pre=pre: ops.shared_prefix_attention(q, kv, batch, pre)))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 2]):
            got.append((i % 3, calls[i % 3]()))
    torch.cuda.synchronize()
    for i, g in got:
        assert torch.equal(g, want[i])


def test_other_stream(gpu):
    from deltaattention_amd import ops
    announce("paged attention on another stream")
    w = World([1, 50, 1], [3000, 9, 77], 8, 2, 128, 16, "bf16")
    kv, batch, q = ops.PagedKV(w.k.cuda(), w.v.cuda()), w.batch(ops), w.q.cuda()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [w.call(ops, q, kv, batch) for _ in range(4)]
    main = w.call(ops, q, kv, batch)
    side.synchronize()
    w.check(main)
    for g in got:
        assert torch.equal(g, main)


def test_far_pages(gpu):
    """A pool of more than 2^31 elements: offsets past 32 bits."""
    from deltaattention_amd import ops
    announce("paged attention, pool past 32-bit offsets")
    D, page, H = 128, 16, 8
    P = (1 << 31) // (D * page * H) + 4096  # 2^31 elements and more, 4 GiB and more each
    k, v = (torch.zeros(P, H, page, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    gen = torch.Generator().manual_seed(1)
    ids = [P - 1, 5, P - 4000, P - 2, 17, P - 77]
    small_k, small_v = (torch.randn(len(ids), H, page, D, generator=gen).to(torch.bfloat16) for _ in range(2))
    at = torch.tensor(ids).cuda()
    k[at], v[at] = small_k.cuda(), small_v.cuda()
    table = _i([ids[:4], ids[2:]])
    for new in ([1, 1], [40, 1]):
        cu = _cu(new)
        q = torch.randn(cu[-1], 32, D, generator=gen).to(torch.bfloat16)
        lengths = [60, 64]
        got = ops.paged_attention(q.cuda(), ops.PagedKV(k, v), ops.PagedBatch(table, _i(lengths), cu))
        want, tol = R.attention(q, small_k, small_v, [[0, 1, 2, 3], [2, 3, 4, 5]], lengths, cu)
        close(got, want, tol)
    x = torch.randn(1, H, D, generator=gen).to(torch.bfloat16)
    ops.append_paged(ops.PagedKV(k, v), ops.PagedBatch(table[:1], _i([4])), x.cuda(), x.cuda())
    assert torch.equal(k[P - 1, :, 3].cpu(), x[0]) and torch.equal(v[P - 1, :, 3].cpu(), x[0])
