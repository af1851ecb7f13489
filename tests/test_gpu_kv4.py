"""Rows in 4 bits, eviction by accumulated weight and decode attention over 4-bit rows against
plain restatements in 64 bits (tests/kv4_reference.py), at the sizes, types and masks where
they can go wrong."""
import math

import pytest
import torch

import kv4_reference as ref
from conftest import announce

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(gen, *shape):
    """Rows whose groups span many powers of two, with some elements exactly on rounding borders."""
    x = torch.randn(*shape, generator=gen) * torch.exp(2.0 * torch.randn(*shape[:-1], 1, generator=gen))
    edge = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -5.0, 0.0, -0.0])
    pick = torch.randint(0, 12, shape, generator=gen)
    return torch.where(torch.rand(shape, generator=gen) < 0.2, edge[pick], x)


def _cache(gpu, gen, B, H, cap, D, lengths, zero_counts=True):
    """A cache of random rows on the GPU and the same on the CPU in 64 bits; rows past a head's
    length and rows of count 0 hold the bytes of NaN and of the largest power."""
    from deltaattention_amd import ops
    G = ref.groups(D)
    kc, ks = ref.encode(torch.randn(B, H, cap, D, generator=gen) * torch.exp(0.7 * torch.randn(B, H, 1, D, generator=gen)))
    vc, vs = ref.encode(torch.randn(B, H, cap, D, generator=gen))
    counts = torch.randint(1, 9, (B, H, cap), generator=gen, dtype=torch.int32)
    if zero_counts:
        counts[torch.rand(B, H, cap, generator=gen) < 0.1] = 0
        counts[torch.rand(B, H, cap, generator=gen) < 0.02] = -3
    lens = torch.tensor(lengths, dtype=torch.int32).view(B, H)
    dead = (counts <= 0) | (torch.arange(cap) >= lens[..., None])
    for sc in (ks, vs):
        sc[dead] = torch.where(torch.rand(B, H, cap, G, generator=gen) < 0.5, 255, 254)[dead].to(torch.uint8)
    mass = torch.rand(B, H, cap, generator=gen)
    ts = (torch.arange(cap, dtype=torch.int32) * 3).expand(B, H, cap).contiguous()
    kv = ops.KV4(kc.to(gpu), ks.to(gpu), vc.to(gpu), vs.to(gpu), counts.to(gpu), ts.to(gpu), lens.to(gpu), D,
                 mass.to(gpu))
    return kv, (ref.decode(kc, ks, D), ref.decode(vc, vs, D), counts, lens, mass)


# ---- rows into 4 bits and back --------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,H,N,D", [(1, 1, 1, 8), (2, 3, 7, 40), (1, 2, 65, 64), (3, 1, 33, 80), (1, 4, 130, 96),
                                     (2, 2, 257, 128), (1, 1, 5, 120)])
def test_quantize(gpu, B, H, N, D, dtype):
    from deltaattention_amd import ops
    announce(f"quantize {B}x{H}x{N}x{D} {dtype}")
    gen = _gen(B * 1000 + N + D)
    k, v = (_rows(gen, B, N, H, D).to(DTYPES[dtype]).transpose(1, 2) for _ in range(2))
    kv = ops.quantize_kv4(k.to(gpu), v.to(gpu))
    for x, codes, scales in ((k, kv.k_codes, kv.k_scales), (v, kv.v_codes, kv.v_scales)):
        want_c, want_s = ref.encode(x)
        assert torch.equal(scales.cpu(), want_s)
        assert torch.equal(codes.cpu(), want_c)
    assert (kv.counts == 1).all() and (kv.mass == 0).all() and (kv.lengths == N).all()
    assert torch.equal(kv.timestamps.cpu(), torch.arange(N, dtype=torch.int32).expand(B, H, N))
    for out in DTYPES.values():
        for x, codes, scales in zip(ops.dequantize_kv4(kv, out), (kv.k_codes, kv.v_codes), (kv.k_scales, kv.v_scales)):
            assert x.dtype == out
            # one rounding to the output type (bf16 and fp32 hold every value)
            assert torch.equal(x.cpu(), ref.decode(codes, scales, D).to(out))


def test_quantize_extremes(gpu):
    """Zeros, the smallest and largest magnitudes, and groups that hold an infinity or a NaN."""
    from deltaattention_amd import ops
    x = torch.zeros(1, 1, 9, 64)
    x[0, 0, 1, 3] = 1e-45
    x[0, 0, 2, :] = torch.linspace(-3e38, 3e38, 64)
    x[0, 0, 3, 5] = math.inf
    x[0, 0, 4, 40] = math.nan
    x[0, 0, 5, 1] = -math.inf
    x[0, 0, 6, :32] = 6.0
    x[0, 0, 7, :32] = 6.0000005
    x[0, 0, 8, :] = torch.linspace(-3e38, 3e38, 64, dtype=torch.float64).float()
    announce("quantize extremes")
    kv = ops.quantize_kv4(x.to(gpu), x.to(gpu))
    want_c, want_s = ref.encode(x)
    assert torch.equal(kv.k_scales.cpu(), want_s) and torch.equal(kv.v_codes.cpu(), want_c)
    assert [int(s) for s in kv.k_scales[0, 0, 3].cpu()] == [255, 2]
    back = ops.dequantize_kv4(kv, torch.float32)[0].cpu()
    assert torch.isnan(back[0, 0, 3, :32]).all() and torch.isnan(back[0, 0, 4, 32:]).all()
    # row 2's own step, 6e38 / 63, passes fp32's largest number: it holds what linspace makes of that
    assert torch.isfinite(back[0, 0, [0, 1, 6, 7, 8]]).all() and (back[0, 0, 3, 32:] == 0).all()
    assert torch.equal(torch.isfinite(back).view(9, 2, 32).all(-1), torch.isfinite(x).view(9, 2, 32).all(-1))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_quantize_index_lengths(gpu, dtype):
    """Chosen rows with their counts, positions and mass; rows past the length and rows that are
    not there come out zero, and rows behind the last chosen stay as they were."""
    from deltaattention_amd import ops
    B, H, N, D, M, cap = 2, 3, 50, 72, 21, 24
    gen = _gen(5)
    k, v = (_rows(gen, B, H, N, D).to(DTYPES[dtype]) for _ in range(2))
    counts = torch.randint(1, 9, (B, H, N), generator=gen, dtype=torch.int32)
    ts = torch.randint(0, 999, (B, H, N), generator=gen, dtype=torch.int32)
    mass = torch.rand(B, H, N, generator=gen)
    index = torch.stack([torch.randperm(N, generator=gen)[:M].sort().values for _ in range(B * H)]).view(B, H, M).int()
    index[0, 0, 4], index[1, 2, 7], index[1, 1, 0] = -1, N, 2 ** 31 - 1
    lens = torch.tensor([[M, 0, 1], [M + 5, 20, -4]], dtype=torch.int32)
    announce("quantize index")
    kv = ops.quantize_kv4(k.to(gpu), v.to(gpu), counts.to(gpu), ts.to(gpu), mass.to(gpu), lens.to(gpu), index.to(gpu),
                          capacity=cap)
    n = lens.clamp(0, M)
    assert torch.equal(kv.lengths.cpu(), n)
    live = (torch.arange(M) < n[..., None]) & (index >= 0) & (index < N)
    at = index.long().clamp(0, N - 1)
    at = torch.where((index >= 0) & (index < N), at, 0)
    for got, src in ((kv.counts, counts), (kv.timestamps, ts), (kv.mass, mass)):
        want = torch.where(live, torch.gather(src, 2, at), torch.zeros((), dtype=src.dtype))
        assert torch.equal(got[:, :, :M].cpu(), want)
    for got_c, got_s, x in ((kv.k_codes, kv.k_scales, k), (kv.v_codes, kv.v_scales, v)):
        want_c, want_s = ref.encode(torch.gather(x, 2, at[..., None].expand(B, H, M, D)))
        assert torch.equal(got_c[:, :, :M].cpu(), torch.where(live[..., None], want_c, torch.zeros((), dtype=torch.uint8)))
        assert torch.equal(got_s[:, :, :M].cpu(), torch.where(live[..., None], want_s, torch.zeros((), dtype=torch.uint8)))
    rows = ops.dequantize_kv4(kv, torch.float32, rows=M)[0].cpu()
    assert (rows[~live] == 0).all()


# ---- the rows a budget leaves -----------------------------------------------------------------


HEAVY = [  # N, lengths, budget, sinks, recent
    (1, [1, 0, 1, 1], 1, 0, 0), (5, [5, 4, 3, 0], 3, 1, 1), (64, [64, 63, 17, 1], 16, 4, 8), (65, [65] * 4, 64, 0, 64),
    (1023, [1023, 1000, 900, 3], 500, 4, 64), (1025, [1025, 1024, 1025, 501], 500, 0, 0),
    (3001, [3001, 2999, 1500, 2000], 1500, 16, 256), (5000, [5000, 4097, 4999, 40], 77, 77, 0),
    (5000, [5000, 4097, 4999, 40], 78, 0, 77), (20000, [20000, 19999, 12345, 20000], 7001, 4, 1000),
    (140001, [140001, 131073, 99999, 140001], 30011, 4, 1000),
]


@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
@pytest.mark.parametrize("N,lengths,budget,sinks,recent", HEAVY, ids=[f"N{c[0]}-b{c[2]}-{c[3]}-{c[4]}" for c in HEAVY])
def test_heavy_rows(gpu, N, lengths, budget, sinks, recent, kind):
    from deltaattention_amd import ops
    gen = _gen(N + budget)
    if kind == "spread":
        mass = torch.exp(4 * torch.randn(2, 2, N, generator=gen) - 5)
    elif kind == "ties":  # most rows without any weight, the others of a few values
        mass = torch.randint(0, 3, (2, 2, N), generator=gen).float() * (torch.rand(2, 2, N, generator=gen) < 0.3)
    else:  # negative numbers, both zeros, infinities, the smallest numbers
        pool = torch.tensor([0.0, -0.0, -1.0, 1.0, math.inf, -math.inf, 1e-45, -1e-45, 3e38, 1.0000001])
        mass = pool[torch.randint(0, 10, (2, 2, N), generator=gen)]
    lens = torch.tensor(lengths, dtype=torch.int32).view(2, 2)
    announce(f"heavy {kind} N={N} budget={budget}")
    index, kept = ops.heavy_rows(mass.to(gpu), budget, sinks, recent, lengths=lens.to(gpu))
    index, kept = index.cpu(), kept.cpu()
    for b in range(2):
        for h in range(2):
            want = ref.heavy(mass[b, h].tolist(), int(lens[b, h]), budget, sinks, recent)
            assert int(kept[b, h]) == len(want)
            assert index[b, h].tolist() == want + [-1] * (budget - len(want))


@pytest.mark.parametrize("D", [8, 64, 88, 128])
@pytest.mark.parametrize("cap,lengths,budget,sinks,recent,room", [
    (9, [9, 0, 1, 8], 4, 1, 1, 4), (40, [40, 39, 12, 11], 12, 0, 3, 20), (700, [700, 699, 128, 0], 127, 4, 64, 127),
    (33, [33, 2, 40, -1], 60, 4, 8, 64), (600, [600, 599, 257, 0], 257, 4, 64, 300),
    (5000, [5000, 4097, 256, 255], 256, 0, 1, 256), (17000, [17000, 100, 16999, 99], 99, 3, 4, 100)])
def test_evict(gpu, D, cap, lengths, budget, sinks, recent, room):
    from deltaattention_amd import ops
    gen = _gen(cap + D)
    kv, (_, _, counts, lens, mass) = _cache(gpu, gen, 2, 2, cap, D, lengths)
    kept_before = {n: getattr(kv, n).clone() for n in ("k_codes", "k_scales", "v_codes", "v_scales", "counts", "mass")}
    announce(f"evict D={D} cap={cap} budget={budget}")
    new = ops.evict_kv4(kv, budget, sinks, recent, capacity=room)
    assert new.capacity == room
    for name, t in kept_before.items():  # the old cache stays as it is
        assert torch.equal(getattr(kv, name), t)
    for b in range(2):
        for h in range(2):
            n = min(max(int(lens[b, h]), 0), cap)
            rows = ref.heavy(mass[b, h].tolist(), n, budget, sinks, recent)
            assert int(new.lengths[b, h]) == len(rows)
            at = torch.tensor(rows, dtype=torch.long)
            for name in ("k_codes", "k_scales", "v_codes", "v_scales", "counts", "timestamps", "mass"):
                got, src = getattr(new, name)[b, h].cpu(), getattr(kv, name)[b, h].cpu()
                assert torch.equal(got[:len(rows)], src[at]), name
                assert (got[len(rows):budget] == 0).all(), name


@pytest.mark.parametrize("cap,budget", [(700, 200), (700, 400), (17000, 200)])
def test_evict_index(gpu, cap, budget):
    """The rows' numbers that the C entry point gives back are heavy_rows'."""
    from deltaattention_amd import ops
    from deltaattention_amd._native import call_on, lib
    kv, _ = _cache(gpu, _gen(cap + budget), 1, 3, cap, 64, [cap, cap - 3, budget - 1])
    want, kept = ops.heavy_rows(kv.mass, budget, 4, 16, lengths=kv.lengths)
    out = ops.KV4.empty(1, 3, budget, 64, gpu)
    index = torch.empty(1, 3, budget, dtype=torch.int32, device=gpu)
    n = lib().da_kv4_evict_workspace_size(1, 3, cap, budget)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device=gpu)
    announce(f"evict index cap={cap} budget={budget}")
    assert call_on(out.device, lib().da_kv4_evict, kv._ref, 1, 3, 64, budget, 4, 16, out._ref, index.data_ptr(),
                   ws.data_ptr() if n else None, n) == 0
    assert torch.equal(index, want) and torch.equal(out.lengths, kept)


# ---- decode attention ---------------------------------------------------------------------------


ATTEND = [  # B, H, G, D, cap, lengths, W, exact, dtype
    (1, 1, 1, 8, 1, [1], 1, 0, "bf16"), (1, 1, 1, 128, 1, [0], 1, 1, "bf16"), (1, 2, 4, 128, 64, [64, 31], 16, 16, "bf16"),
    (2, 2, 4, 128, 200, [200, 0, 33, 129], 50, 50, "bf16"), (1, 2, 1, 64, 513, [513, 512], 64, 17, "fp16"),
    (1, 3, 7, 80, 333, [333, 1, 32], 128, 100, "fp16"), (1, 1, 16, 40, 1000, [1000], 33, 33, "bf16"),
    (1, 1, 17, 96, 700, [699], 20, 20, "bf16"), (1, 1, 64, 64, 300, [300], 5, 5, "fp32"),
    (2, 1, 8, 128, 777, [776, 5], 128, 128, "fp32"), (1, 2, 4, 24, 100, [100, 99], 0, 0, "fp32"),
    (1, 8, 4, 128, 4100, [4100, 4099, 4096, 3000, 2049, 128, 127, 0], 128, 128, "bf16"),
    (1, 1, 4, 128, 70001, [69999], 64, 64, "fp16"), (5, 3, 2, 56, 97, list(range(0, 98, 7)) + [97], 3, 2, "bf16"),
    (1, 1, 4, 128, 140000, [139999], 64, 64, "bf16"), (1, 2, 2, 64, 140000, [0, 5], 16, 16, "fp32"),
]


def _ids(c):
    return f"B{c[0]}H{c[1]}G{c[2]}D{c[3]}-cap{c[4]}-W{c[6]}.{c[7]}-{c[8]}"


def _attend_want(q, parts, kx, vx, exact, G):
    """Per (b, h): out, its bound, the rows' weights and their bound."""
    kf, vf, counts, lens, mass = parts
    for b in range(q.shape[0]):
        for h in range(kf.shape[1]):
            n = min(max(int(lens[b, h]), 0), kf.shape[2])
            k = torch.cat([kf[b, h, :n], kx[b, h, :exact].double()])
            v = torch.cat([vf[b, h, :n], vx[b, h, :exact].double()])
            size = torch.cat([counts[b, h, :n].clamp(min=0).double(), torch.ones(exact).double()])
            out, w, spread, drift = ref.attention(q[b, h * G:(h + 1) * G].double(), k, v, size)
            # weights enter the product in parts of 2^-17 (16-bit outputs) or less; sums of n + exact
            # terms in fp32; the output's own rounding is half a step
            eps = torch.finfo(q.dtype).eps / 2
            rel = drift[:, None] + 2.0 ** -16 * (q.dtype != torch.float32) + (n + exact + 64) * 2.0 ** -24
            tol = eps * out.abs() + (1 + eps) * rel * spread + 1e-30
            wsum = w[:, :n].sum(0)
            wtol = (w[:, :n] * (drift[:, None] + (n + exact + 64) * 2.0 ** -24)).sum(0) + 2.0 ** -23 * (wsum + mass[b, h, :n].double())
            yield b, h, n, out, tol, wsum, wtol


@pytest.mark.parametrize("c", ATTEND, ids=[_ids(c) for c in ATTEND])
@pytest.mark.parametrize("accumulate", [False, True])
def test_attend(gpu, c, accumulate):
    from deltaattention_amd import ops
    B, H, G, D, cap, lengths, W, exact, dtype = c
    gen = _gen(cap + D + W)
    kv, parts = _cache(gpu, gen, B, H, cap, D, lengths)
    dt = DTYPES[dtype]
    q = (1.5 * torch.randn(B, H * G, D, generator=gen)).to(dt)
    kx, vx = (torch.randn(B, H, W, D, generator=gen).to(dt) for _ in range(2))
    kx[:, :, exact:], vx[:, :, exact:] = math.nan, math.inf  # slots not in use
    ring = (kx.to(gpu), vx.to(gpu), exact) if W else (None, None, None)
    announce(f"attend {_ids(c)} accumulate={accumulate}")
    out = ops.decode_attention_kv4(q.to(gpu).unsqueeze(2), kv, *ring, accumulate=accumulate).cpu()
    mass = kv.mass.cpu()
    assert out.shape == (B, H * G, 1, D) and out.dtype == dt
    for b, h, n, want, tol, wsum, wtol in _attend_want(q, parts, kx, vx, exact, G):
        got = out[b, h * G:(h + 1) * G, 0].double()
        assert ((got - want).abs() <= tol).all(), f"({b}, {h}): {((got - want).abs() / tol).max():.3g} of the bound"
        before = parts[4][b, h]
        if accumulate:
            off = (mass[b, h, :n].double() - before[:n].double() - wsum).abs()
            assert (off <= wtol).all(), f"({b}, {h}): weights {(off / wtol).max():.3g} of the bound"
            assert torch.equal(mass[b, h, n:], before[n:])  # rows behind the length stay
        else:
            assert torch.equal(mass[b, h], before)


def test_attend_strided(gpu):
    """q, the ring and the output as views: heads inside a wider row, a ring cut out of a longer one."""
    from deltaattention_amd import ops
    B, H, G, D, cap, W = 2, 2, 4, 128, 150, 40
    gen = _gen(77)
    kv, parts = _cache(gpu, gen, B, H, cap, D, [150, 149, 3, 77])
    wide = (1.5 * torch.randn(B, 1, H * G, D + 8, generator=gen)).bfloat16()
    q = wide.to(gpu)[..., 3:D + 3].transpose(1, 2)  # rows not 16-byte aligned
    rk, rv = (torch.randn(B, W + 9, H, D, generator=gen).bfloat16() for _ in range(2))
    kx, vx = (x.to(gpu)[:, 5:5 + W].transpose(1, 2) for x in (rk, rv))
    out = torch.zeros(B, 1, H * G + 1, D, dtype=torch.bfloat16, device=gpu)
    announce("attend strided")
    got = ops.decode_attention_kv4(q, kv, kx, vx, out=out[:, :, :H * G].transpose(1, 2))
    assert got.data_ptr() == out.data_ptr() and (out[:, :, H * G] == 0).all()
    same = ops.decode_attention_kv4(q.contiguous(), kv, kx.contiguous(), vx.contiguous())
    assert torch.equal(got, same)
    qc = wide[..., 3:D + 3].transpose(1, 2).squeeze(2)
    for b, h, n, want, tol, _, _ in _attend_want(qc, parts, rk[:, 5:5 + W].transpose(1, 2), rv[:, 5:5 + W].transpose(1, 2), W, G):
        assert ((got[b, h * G:(h + 1) * G, 0].cpu().double() - want).abs() <= tol).all()


def test_attend_all_masked(gpu):
    """No row in use and no ring, or rows of count 0 alone: zeros, and no weight anywhere."""
    from deltaattention_amd import ops
    gen = _gen(3)
    kv, _ = _cache(gpu, gen, 1, 2, 40, 64, [0, 40])
    kv.counts.zero_()
    before = kv.mass.clone()
    q = torch.randn(1, 8, 1, 64, generator=gen).to(gpu)
    announce("attend masked")
    assert (ops.decode_attention_kv4(q, kv, accumulate=True) == 0).all()
    assert torch.equal(kv.mass, before)


def test_attend_nan_is_seen(gpu):
    """A live row that reads back as NaN is not hidden."""
    from deltaattention_amd import ops
    gen = _gen(4)
    kv, _ = _cache(gpu, gen, 1, 1, 40, 64, [40], zero_counts=False)
    kv.k_scales[0, 0, 7, 0] = 255
    q = torch.randn(1, 4, 1, 64, generator=gen).bfloat16().to(gpu)
    announce("attend nan")
    assert torch.isnan(ops.decode_attention_kv4(q, kv)).all()


# ---- streams and graphs -----------------------------------------------------------------------------


def _chain(ops, s):
    """The operators as a program runs them: the prompt's weights, the rows they leave in 4 bits, a
    token over those, and a second cut."""
    mass = ops.attention_mass(s["q"], s["k"])
    index, kept = ops.heavy_rows(mass, 40, 2, 8)
    kv = ops.quantize_kv4(s["k"], s["v"], mass=mass, index=index, lengths=kept)
    out = ops.decode_attention_kv4(s["q"][:, :, -1:], kv, s["k"][:, :, -16:], s["v"][:, :, -16:], accumulate=True)
    small = ops.evict_kv4(kv, 24, 2, 8)
    k, v = ops.dequantize_kv4(small)
    return [mass, index, kept, out, kv.mass, small.mass, small.timestamps, small.lengths, k, v]


def _chain_inputs(gpu, seed, B=2, H=2, G=4, N=300, D=128):
    gen = _gen(seed)
    return {"q": torch.randn(B, H * G, 48, D, generator=gen).bfloat16().to(gpu),
            "k": torch.randn(B, H, N, D, generator=gen).bfloat16().to(gpu),
            "v": torch.randn(B, H, N, D, generator=gen).bfloat16().to(gpu)}


def test_chain_stream_and_graph(gpu):
    """The chain on a stream of its own and captured into a graph gives, replay after replay and with
    eager work and other inputs between, what it gives eagerly."""
    from deltaattention_amd import ops
    announce("kv4 chain: eager, side stream, graph")
    a, b = _chain_inputs(gpu, 1), _chain_inputs(gpu, 2)
    want_a, want_b = ([t.clone() for t in _chain(ops, s)] for s in (a, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _chain(ops, a)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for x, y in zip(got, want_a):
        assert torch.equal(x, y)
    s = {n: t.clone() for n, t in a.items()}
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _chain(ops, s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _chain(ops, s)
    for turn in range(4):
        src, want = ((a, want_a), (b, want_b))[turn % 2]
        for n, t in src.items():
            s[n].copy_(t)
        graph.replay()
        for x, y in zip(held, want):
            assert torch.equal(x, y), turn
        for x, y in zip(_chain(ops, b), want_b):  # eager work between the replays
            assert torch.equal(x, y)
        torch.cuda.synchronize()


def test_two_streams_at_once(gpu):
    """Two programs with their own inputs on two streams do not disturb each other."""
    from deltaattention_amd import ops
    announce("kv4 two streams")
    ins = [_chain_inputs(gpu, 3 + i, N=2000) for i in range(2)]
    want = [[t.clone() for t in _chain(ops, s)] for s in ins]
    streams = [torch.cuda.Stream() for _ in ins]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = _chain(ops, ins[i])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for x, y in zip(g, w):
            assert torch.equal(x, y)


def test_deterministic(gpu):
    """The same call gives the same bits, splits and all."""
    from deltaattention_amd import ops
    gen = _gen(12)
    q = torch.randn(1, 8, 700, 64, generator=gen).to(gpu)
    k = torch.randn(1, 2, 5000, 64, generator=gen).to(gpu)
    kv, _ = _cache(gpu, gen, 1, 2, 9000, 64, [9000, 8000])
    mass = kv.mass.clone()
    announce("kv4 deterministic")
    first = None
    for _ in range(3):
        kv.mass.copy_(mass)
        got = [ops.attention_mass(q, k), ops.decode_attention_kv4(q[:, :, :1], kv, accumulate=True), kv.mass.clone()]
        if first is not None:
            for x, y in zip(got, first):
                assert torch.equal(x, y)
        first = got
