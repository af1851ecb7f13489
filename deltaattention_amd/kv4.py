"""A decode cache that stays bounded: rows in 4 bits, the attention weight each row received,
eviction by it, and decode attention over 4-bit rows (include/deltaattn_cache.h).

The compressed cache of the reference (deltaDecoding.py:111-233) keeps every anchor at full
width; these operations have no counterpart there.  They follow ``ops``: GPU tensors, the
current stream of the tensors' device, no synchronisation, no CPU fallback, errors as
Python exceptions.  Users reach them as ``ops.KV4``, ``ops.attention_mass`` and so on;
``deltaDecoding.FourBitCompressedCache`` is the cache object built on them.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional, Tuple

import torch

from ._native import Kv4Block, call_on, check, dtype_code, lib

__all__ = ["KV4", "attention_mass", "heavy_rows", "quantize_kv4", "dequantize_kv4", "evict_kv4",
           "decode_update_kv4", "decode_attention_kv4"]

_I32, _F32, _U8 = torch.int32, torch.float32, torch.uint8


def _want(t: torch.Tensor, name: str, shape, dtype, device) -> None:
    """Refuse a tensor that is not contiguous, of this shape and type and on this device."""
    if t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.device == device:
        return
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {list(shape)}, got {list(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    raise ValueError(f"{name} must be contiguous")


def _gpu(t: torch.Tensor, name: str) -> torch.device:
    if t.device.type != "cuda":
        raise ValueError(f"deltaattention_amd operations take GPU tensors ({name} is on {t.device}); "
                         "there is no CPU path")
    return t.device


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with a contiguous head dimension and rows that begin at multiples of 16 bytes."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():  # a head dimension is a multiple of 8 elements
            return t
        per = 4 if t.dtype == _F32 else 8
        s = t.stride()
        if s[-1] == 1 and not any(x % per for x, n in zip(s[:-1], t.shape) if n > 1):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t: torch.Tensor):
    """Batch, head and row strides; 0 for a dimension of one, whose stride means nothing."""
    return [s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape)]


@functools.lru_cache(maxsize=1024)
def _mass_bytes(*shape) -> int:
    return lib().da_attention_mass_workspace_size(*shape)


@functools.lru_cache(maxsize=1024)
def _evict_bytes(*shape) -> int:
    return lib().da_kv4_evict_workspace_size(*shape)


@functools.lru_cache(maxsize=1024)
def _attention_bytes(*shape) -> int:
    return lib().da_kv4_attention_workspace_size(*shape)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


_set = object.__setattr__
_TENSORS = ("k_codes", "k_scales", "v_codes", "v_scales", "counts", "timestamps", "lengths", "mass")


@functools.lru_cache(maxsize=1024)
def _layout(B: int, H: int, cap: int, D: int, mass: bool):
    """One allocation's bytes, its fields' offsets in Kv4Block's order, and each one's view."""
    g, size, at, views = (D + 31) // 32, 0, [], {}
    rows, row_stride = (B, H, cap), (H * cap, cap, 1)
    for name, width, dtype in (("k_codes", 16 * g, _U8), ("k_scales", g, _U8), ("v_codes", 16 * g, _U8),
                               ("v_scales", g, _U8), ("counts", 4, _I32), ("timestamps", 4, _I32),
                               ("lengths", 4, _I32), ("mass", 4, _F32)):
        if name == "mass" and not mass:
            at.append(None)
            views[name] = None
            continue
        at.append(size)
        if dtype == _U8:
            views[name] = dtype, rows + (width,), (H * cap * width, cap * width, width, 1), size
        elif name == "lengths":
            views[name] = dtype, (B, H), (H, 1), size // 4
        else:
            views[name] = dtype, rows, row_stride, size // 4
        size += (B * H * (1 if name == "lengths" else cap) * width + 255) & ~255
    return size, at, views


class KV4:
    """Key and value rows of one layer in 4 bits, for every (sequence, KV head).

    A row of ``head_dim`` dims is cut into groups of 32; a group has one power of two and
    elements 0, 0.5, 1, 1.5, 2, 3, 4 or 6 times it, with a sign.  ``k_codes`` / ``v_codes``
    [B, Hkv, capacity, 16 * groups] uint8 hold two elements a byte (even dim low),
    ``k_scales`` / ``v_scales`` [B, Hkv, capacity, groups] uint8 the exponents plus 127 (255:
    a group that held an infinity or NaN, which reads back as NaN).  ``counts`` and
    ``timestamps`` [B, Hkv, capacity] int32 are those of the packed anchors (a row of count c
    weighs like c keys), ``mass`` [B, Hkv, capacity] float32 (or None) the attention weight
    each row has received, ``lengths`` [B, Hkv] int32 the rows in use.  All contiguous; the
    tensors of an object are fixed, their contents are not.
    """

    __slots__ = ("k_codes", "k_scales", "v_codes", "v_scales", "counts", "timestamps", "lengths", "mass",
                 "batch", "kv_heads", "capacity", "head_dim", "device", "_block", "_ref", "_own")

    def __init__(self, k_codes, k_scales, v_codes, v_scales, counts, timestamps, lengths, head_dim, mass=None):
        D = int(head_dim)
        if D <= 0 or D > 128 or D % 8:
            raise ValueError(f"head_dim must be a multiple of 8 in [8, 128], got {head_dim}")
        groups = (D + 31) // 32
        if k_codes.dim() != 4:
            raise ValueError("k_codes must have shape [B, Hkv, capacity, 16 * groups]")
        device = _gpu(k_codes, "k_codes")
        B, H, cap, _ = k_codes.shape
        if not (B and H and cap):
            raise ValueError("a cache needs sequences, heads and rows")
        wide, narrow, rows = (B, H, cap, 16 * groups), (B, H, cap, groups), (B, H, cap)
        _want(k_codes, "k_codes", wide, _U8, device)
        _want(v_codes, "v_codes", wide, _U8, device)
        _want(k_scales, "k_scales", narrow, _U8, device)
        _want(v_scales, "v_scales", narrow, _U8, device)
        _want(counts, "counts", rows, _I32, device)
        _want(timestamps, "timestamps", rows, _I32, device)
        _want(lengths, "lengths", (B, H), _I32, device)
        if mass is not None:
            _want(mass, "mass", rows, _F32, device)
        kc, vc, ks, vs = k_codes.data_ptr(), v_codes.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr()
        if (kc | vc) % 16 or (ks | vs) % 4:
            raise ValueError("codes must be 16-byte aligned, scales 4-byte")
        self._put(B, H, cap, D, device, Kv4Block(
            kc, ks, vc, vs, counts.data_ptr(), timestamps.data_ptr(), lengths.data_ptr(),
            None if mass is None else mass.data_ptr(), cap), None)
        _set(self, "k_codes", k_codes)
        _set(self, "k_scales", k_scales)
        _set(self, "v_codes", v_codes)
        _set(self, "v_scales", v_scales)
        _set(self, "counts", counts)
        _set(self, "timestamps", timestamps)
        _set(self, "lengths", lengths)
        _set(self, "mass", mass)

    def _put(self, B, H, cap, D, device, block, own):
        _set(self, "batch", B)
        _set(self, "kv_heads", H)
        _set(self, "capacity", cap)
        _set(self, "head_dim", D)
        _set(self, "device", device)
        _set(self, "_block", block)
        _set(self, "_ref", ctypes.byref(block))
        _set(self, "_own", own)

    def __setattr__(self, name, value):
        raise AttributeError(f"KV4.{name} is fixed; build another KV4 from the tensors")

    @classmethod
    def empty(cls, batch: int, kv_heads: int, capacity: int, head_dim: int, device="cuda", mass: bool = True) -> "KV4":
        """A cache of ``capacity`` rows a head with undefined contents (``lengths`` too), in one
        allocation; its tensors are views that are made when they are first asked for."""
        B, H, cap, D = int(batch), int(kv_heads), int(capacity), int(head_dim)
        if not (B > 0 and H > 0 and cap > 0) or D <= 0 or D > 128 or D % 8:
            raise ValueError(f"no cache of {batch} sequences, {kv_heads} heads, {capacity} rows and head_dim {head_dim}")
        return cls._over(torch.empty((_layout(B, H, cap, D, bool(mass))[0],), dtype=_U8, device=device), B, H, cap, D,
                         bool(mass))

    @classmethod
    def _over(cls, own, B, H, cap, D, mass):
        """The cache whose fields lie in the bytes ``own`` (_layout)."""
        size, at, views = _layout(B, H, cap, D, mass)
        device, p = _gpu(own, "the cache"), own.data_ptr()
        if own.shape != (size,) or p % 256:
            raise ValueError(f"{size} bytes at a multiple of 256 expected, got {list(own.shape)}")
        self = cls.__new__(cls)
        self._put(B, H, cap, D, device, Kv4Block(*[None if x is None else p + x for x in at], cap),
                  (views, {_U8: own}))
        return self

    def __getattr__(self, name):
        # only for what is not there yet: a tensor of a cache that empty() made
        if name not in _TENSORS:
            raise AttributeError(name)
        views, own = self._own
        view = views[name]
        if view is None:  # a cache without mass
            t = None
        else:
            dtype, shape, stride, first = view
            base = own.get(dtype)
            if base is None:
                base = own[dtype] = own[_U8].view(dtype)
            t = base.as_strided(shape, stride, first)
        _set(self, name, t)
        return t

    def clone(self) -> "KV4":
        """A copy in memory of its own (of the rows past the lengths too)."""
        out = KV4.empty(self.batch, self.kv_heads, self.capacity, self.head_dim, self.device, self.mass is not None)
        for name in _TENSORS:
            t = getattr(self, name)
            if t is not None:
                getattr(out, name).copy_(t)
        return out

    def __deepcopy__(self, memo):
        return self.clone()

    def __reduce__(self):
        # copy.copy: another KV4 of the same tensors; pickling: of the tensors as torch pickles them
        if self._own:  # one allocation: its bytes, not eight views of them
            return KV4._over, (self._own[1][_U8], self.batch, self.kv_heads, self.capacity, self.head_dim,
                               self._own[0]["mass"] is not None)
        return KV4, (self.k_codes, self.k_scales, self.v_codes, self.v_scales, self.counts, self.timestamps, self.lengths,
                     self.head_dim, self.mass)

    def record_stream(self, stream: torch.cuda.Stream) -> None:
        """``torch.Tensor.record_stream`` of the cache's memory: once the object is gone, it is not
        given out again before what ``stream`` has been given by then is done."""
        for t in [self._own[1][_U8]] if self._own else [getattr(self, name) for name in _TENSORS]:
            if t is not None:
                t.record_stream(stream)


def attention_mass(q: torch.Tensor, k: torch.Tensor, counts: Optional[torch.Tensor] = None,
                   timestamps: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                   q_start: Optional[int] = None, scale: Optional[float] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The attention weight every key receives from the queries: float32 [B, Hkv, Nk], summed over
    the queries and the query heads of each KV head's group.

    q [B, Hq, Nq, D] (usually the prompt's last queries, or all of them), k [B, Hkv, Nk, D].
    Query i is at position ``q_start + i`` (default Nk - Nq, the last ones; needed with
    ``timestamps``) and sees key j if j is below the head's ``lengths`` and its position
    ``timestamps[b, g, j]`` (default j) is not past the query's.  ``counts`` adds log(count) to
    the scores, as packed anchors have it; a count <= 0 hides the key, a timestamp of 2^31 - 1
    too.  A query that sees nothing adds nothing; keys that no query sees, and those past the
    length, get 0, whatever they hold.
    """
    device = _gpu(q, "q")
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q and k are [B, heads, tokens, head_dim]")
    dt = dtype_code(q, k)
    B, Hq, Nq, D = q.shape
    H, N = k.shape[1], k.shape[2]
    if k.device != device or k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"k {list(k.shape)} on {k.device} does not fit q {list(q.shape)} on {device}")
    if not (B and Nq and N and H and Hq) or Hq % H:
        raise ValueError(f"{Hq} query heads over {H} KV heads, {Nq} queries, {N} keys")
    if counts is not None:
        _want(counts, "counts", (B, H, N), _I32, device)
    if timestamps is not None:
        _want(timestamps, "timestamps", (B, H, N), _I32, device)
        if q_start is None:
            raise ValueError("q_start (the position of the first query) is needed with timestamps")
    if lengths is not None:
        _want(lengths, "lengths", (B, H), _I32, device)
    if out is None:
        out = torch.empty((B, H, N), dtype=_F32, device=device)
    else:
        _want(out, "out", (B, H, N), _F32, device)
    q, k = _rows(q), _rows(k)
    n = _mass_bytes(B, Hq, H, Nq, N)
    ws = torch.empty((n,), dtype=_U8, device=device)
    sq, sk = q.stride(), k.stride()
    rc = call_on(device, lib().da_attention_mass, q.data_ptr(), k.data_ptr(), dt, B, Hq, H, Nq, N, D, sq[0], sq[1], sq[2],
                 sk[0], sk[1], sk[2], _ptr(counts), _ptr(timestamps), _ptr(lengths),
                 N - Nq if q_start is None else int(q_start), D ** -0.5 if scale is None else scale, out.data_ptr(),
                 ws.data_ptr(), n)
    check(rc, "da_attention_mass")
    return out


def heavy_rows(mass: torch.Tensor, budget: int, sinks: int = 0, recent: int = 0,
               lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The rows that a budget leaves: mass float32 [B, Hkv, N] -> (index [B, Hkv, budget] int32,
    rows ascending and -1 past them, and their number [B, Hkv] int32).

    A head with at most ``budget`` rows (``lengths``, default N) keeps all.  A longer one keeps
    its first ``sinks`` rows, its last ``recent`` rows, and of those between the
    budget - sinks - recent with the largest mass (a NaN is the largest), ties to the lower row.
    """
    device = _gpu(mass, "mass")
    if mass.dim() != 3:
        raise ValueError("mass is [B, Hkv, N]")
    B, H, N = mass.shape
    _want(mass, "mass", (B, H, N), _F32, device)
    if lengths is not None:
        _want(lengths, "lengths", (B, H), _I32, device)
    budget, sinks, recent = _budget(budget, sinks, recent)
    index = torch.empty((B, H, budget), dtype=_I32, device=device)
    kept = torch.empty((B, H), dtype=_I32, device=device)
    n = _evict_bytes(B, H, N, budget)
    ws = torch.empty((n,), dtype=_U8, device=device) if n else None
    rc = call_on(device, lib().da_heavy_rows, mass.data_ptr(), _ptr(lengths), B, H, N, budget, sinks, recent,
                 index.data_ptr(), kept.data_ptr(), _ptr(ws), n)
    check(rc, "da_heavy_rows")
    return index, kept


def _budget(budget, sinks, recent):
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    if budget <= 0 or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError(f"needs sinks + recent <= budget and a positive budget, got {sinks} + {recent} and {budget}")
    return budget, sinks, recent


def quantize_kv4(k: torch.Tensor, v: torch.Tensor, counts: Optional[torch.Tensor] = None,
                 timestamps: Optional[torch.Tensor] = None, mass: Optional[torch.Tensor] = None,
                 lengths: Optional[torch.Tensor] = None, index: Optional[torch.Tensor] = None,
                 capacity: Optional[int] = None) -> KV4:
    """k, v [B, Hkv, N, D] (any strides) into a new 4-bit cache of ``capacity`` rows a head.

    Without ``index`` row m becomes row m; with it ([B, Hkv, M] int32, as ``heavy_rows`` gives
    it) row index[b, g, m] does.  counts, timestamps and mass [B, Hkv, N] come along (default
    1, the row's number, 0).  ``lengths`` [B, Hkv] are the rows in use (default: all of them);
    rows past them, and those whose index is not a row of k, are zero with count 0, and rows
    from N (M) to the capacity are undefined.
    """
    device = _gpu(k, "k")
    if k.dim() != 4 or v.shape != k.shape or v.device != device:
        raise ValueError("k and v are [B, Hkv, N, D] of one shape on one device")
    dt = dtype_code(k, v)
    B, H, N, D = k.shape
    if not (B and H and N):
        raise ValueError("k and v hold no rows")
    for t, name, ty in ((counts, "counts", _I32), (timestamps, "timestamps", _I32), (mass, "mass", _F32)):
        if t is not None:
            _want(t, name, (B, H, N), ty, device)
    M = N
    if index is not None:
        if index.dim() != 3 or index.shape[2] == 0:
            raise ValueError("index is [B, Hkv, M]")
        M = index.shape[2]
        _want(index, "index", (B, H, M), _I32, device)
    if lengths is not None:
        _want(lengths, "lengths", (B, H), _I32, device)
    capacity = M if capacity is None else int(capacity)
    if capacity < M:
        raise ValueError(f"{M} rows do not fit a capacity of {capacity}")
    k, v = _rows(k), _rows(v)
    out = KV4.empty(B, H, capacity, D, device)
    sk, sv = k.stride(), v.stride()
    rc = call_on(device, lib().da_kv4_quantize, k.data_ptr(), v.data_ptr(), dt, B, H, N, D, sk[0], sk[1], sk[2], sv[0],
                 sv[1], sv[2], _ptr(counts), _ptr(timestamps), _ptr(mass), _ptr(lengths), _ptr(index), M, out._ref)
    check(rc, "da_kv4_quantize")
    return out


def dequantize_kv4(kv: KV4, dtype: torch.dtype = torch.bfloat16, rows: Optional[int] = None):
    """(k, v) [B, Hkv, rows, D]: the values of the first ``rows`` (default: all) 4-bit rows, zero
    past a head's length."""
    N = kv.capacity if rows is None else int(rows)
    if not 0 < N <= kv.capacity:
        raise ValueError(f"rows must lie in [1, {kv.capacity}], got {N}")
    shape = (kv.batch, kv.kv_heads, N, kv.head_dim)
    k, v = (torch.empty(shape, dtype=dtype, device=kv.device) for _ in range(2))
    dt = dtype_code(k)
    rc = call_on(kv.device, lib().da_kv4_dequantize, kv._ref, *shape, k.data_ptr(), v.data_ptr(), dt)
    check(rc, "da_kv4_dequantize")
    return k, v


def evict_kv4(kv: KV4, budget: int, sinks: int = 0, recent: int = 0, capacity: Optional[int] = None) -> KV4:
    """A new cache with the rows of ``kv`` that the budget leaves (the rule of ``heavy_rows`` on
    ``kv.mass`` and ``kv.lengths``), in their order, with their counts, timestamps and mass.
    Rows past those kept are zero up to the budget and undefined from there to ``capacity``
    (default: the budget).  ``kv`` stays as it is."""
    if kv.mass is None:
        raise ValueError("eviction needs the cache's mass")
    budget, sinks, recent = _budget(budget, sinks, recent)
    capacity = budget if capacity is None else int(capacity)
    if capacity < budget:
        raise ValueError(f"a budget of {budget} rows does not fit a capacity of {capacity}")
    B, H, cap, D, device = kv.batch, kv.kv_heads, kv.capacity, kv.head_dim, kv.device
    out = KV4.empty(B, H, capacity, D, device)
    n = _evict_bytes(B, H, cap, budget)
    ws = torch.empty((n,), dtype=_U8, device=device) if n else None
    rc = call_on(device, lib().da_kv4_evict, kv._ref, B, H, D, budget, sinks, recent, out._ref, None, _ptr(ws), n)
    check(rc, "da_kv4_evict")
    return out


def _check_update(kv: KV4, key, value, k_exact, v_exact, k_last, exact_seq_len, total_seq_len) -> int:
    """The type code of ``decode_update_kv4``'s rows, or what it refuses."""
    B, H, D, device = kv.batch, kv.kv_heads, kv.head_dim, kv.device
    dt = dtype_code(key, value, k_exact, v_exact, k_last)
    if key.shape != (B, H, 1, D) or value.shape != key.shape or key.device != device or value.device != device:
        raise ValueError(f"key and value must be {[B, H, 1, D]} on {device}")
    if k_exact.dim() != 4 or not k_exact.shape[2] or k_exact.device != device or v_exact.device != device:
        raise ValueError(f"k_exact and v_exact must be [{B}, {H}, W, {D}] on {device}")
    W = k_exact.shape[2]
    for t, name in ((k_exact, "k_exact"), (v_exact, "v_exact")):
        _want(t, name, (B, H, W, D), k_exact.dtype, device)
    _want(k_last, "k_last", (B, H, D), k_exact.dtype, device)
    if exact_seq_len < 0 or total_seq_len < 0:
        raise ValueError("negative lengths")
    return dt


def decode_update_kv4(kv: KV4, key: torch.Tensor, value: torch.Tensor, k_exact: torch.Tensor, v_exact: torch.Tensor,
                      k_last: torch.Tensor, exact_seq_len: int, total_seq_len: int, threshold: float,
                      use_cosine: bool = False) -> None:
    """One decode token into the ring k_exact, v_exact [B, Hkv, W, D] (slot exact_seq_len % W).  Where
    the ring was full, the token that leaves it merges into its head's last 4-bit row (count + 1) or
    becomes a new one, by the test of ``da_decode_update`` against that row's key as it was
    (k_last [B, Hkv, D], kept up to date).  ``threshold`` is squared for the Euclidean test.  key, value
    [B, Hkv, 1, D], ring and k_last share one type."""
    dt = _check_update(kv, key, value, k_exact, v_exact, k_last, exact_seq_len, total_seq_len)
    B, H, W, D = k_exact.shape
    key, value = _rows(key), _rows(value)
    if _strides(key) != _strides(value):
        key, value = key.contiguous(), value.contiguous()
    sn = _strides(key)
    rc = call_on(kv.device, lib().da_kv4_update, key.data_ptr(), value.data_ptr(), dt, B, H, D, sn[0], sn[1],
                 k_exact.data_ptr(), v_exact.data_ptr(), H * W * D, W * D, D, kv._ref, k_last.data_ptr(),
                 int(exact_seq_len), int(total_seq_len), W, threshold, 1 if use_cosine else 0)
    check(rc, "da_kv4_update")


def _check_query(q: torch.Tensor, kv: KV4) -> Tuple[int, int, int]:
    """(B, Hq, D) of one token's queries over ``kv``."""
    device, H = kv.device, kv.kv_heads
    shape = q.shape
    if len(shape) == 4 and shape[2] == 1:
        B, Hq, _, D = shape
    elif len(shape) == 3:
        B, Hq, D = shape
    else:
        raise ValueError("q is [B, Hq, 1, D] or [B, Hq, D]")
    if q.device != device or B != kv.batch or D != kv.head_dim or Hq % H or not Hq:
        raise ValueError(f"q {list(shape)} on {q.device} does not fit a cache of {kv.batch} sequences, {H} KV heads "
                         f"and head_dim {kv.head_dim} on {device}")
    return B, Hq, D


def decode_attention_kv4(q: torch.Tensor, kv: KV4, k_exact: Optional[torch.Tensor] = None,
                         v_exact: Optional[torch.Tensor] = None, exact_len: Optional[int] = None,
                         scale: Optional[float] = None, accumulate: bool = False,
                         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One decode token: q [B, Hq, 1, D] (or [B, Hq, D]) -> the same shape, attention over the 4-bit
    rows (scores + log(count)) and the first ``exact_len`` (default W) slots of the ring
    k_exact, v_exact [B, Hkv, W, D] in q's type.

    ``accumulate`` adds each row's softmax weight, summed over its group's query heads, to
    ``kv.mass``.  A head without any key gives zeros.  Query head h reads KV head
    h // (Hq // Hkv).
    """
    B, Hq, D = _check_query(q, kv)
    device, H, shape = kv.device, kv.kv_heads, q.shape
    if (k_exact is None) != (v_exact is None):
        raise ValueError("k_exact and v_exact come together")
    if accumulate and kv.mass is None:
        raise ValueError("accumulate needs the cache's mass")
    dt = dtype_code(q, k_exact, v_exact, out)
    sx, W, kx, vx = (0, 0, 0), 0, None, None
    if k_exact is not None:
        xs = k_exact.shape
        if len(xs) != 4 or xs[0] != B or xs[1] != H or xs[3] != D or v_exact.shape != xs or k_exact.device != device \
                or v_exact.device != device:
            raise ValueError(f"k_exact and v_exact must be [{B}, {H}, W, {D}] on {device}")
        W = xs[2]
        if W:
            if not (k_exact.is_contiguous() and v_exact.is_contiguous() and (k_exact.data_ptr() | v_exact.data_ptr()) % 16 == 0):
                k_exact, v_exact = _rows(k_exact), _rows(v_exact)
                if _strides(v_exact) != _strides(k_exact):
                    k_exact, v_exact = (t.clone(memory_format=torch.contiguous_format) for t in (k_exact, v_exact))
            sx = k_exact.stride()
        kx, vx = k_exact.data_ptr(), v_exact.data_ptr()
    n_exact = W if exact_len is None else int(exact_len)
    if not 0 <= n_exact <= W:
        raise ValueError(f"exact_len must lie in [0, {W}], got {n_exact}")
    q = _rows(q)
    sq = q.stride()
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=device)
    elif out.shape != shape or out.device != device or out.stride(-1) != 1:
        raise ValueError("out must have q's shape and device and a contiguous head dimension")
    so = out.stride()
    n = _attention_bytes(B, Hq, H, kv.capacity, 1 if accumulate else 0)
    ws = torch.empty((n,), dtype=_U8, device=device) if n else None  # held until the call is on its stream
    rc = call_on(device, lib().da_kv4_attention, q.data_ptr(), dt, B, Hq, H, D, sq[0], sq[1], kv._ref, kx, vx, sx[0],
                 sx[1], sx[2], n_exact, D ** -0.5 if scale is None else scale, 1 if accumulate else 0, out.data_ptr(),
                 so[0], so[1], _ptr(ws), n)
    check(rc, "da_kv4_attention")
    return out
