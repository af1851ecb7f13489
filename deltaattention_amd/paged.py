"""A paged key/value cache at full width: new tokens rotated and written into pages, attention of
new tokens over the pages of their sequences, and the same where groups of sequences share their
first tokens (include/deltaattn_paged.h).

The dense path of the reference keeps no cache (modeling_llama.py:778-803); these operations
have no counterpart there.  They follow ``ops``: GPU tensors, the current stream of the tensors'
device, no synchronisation, no CPU fallback, errors as Python exceptions.  Users reach them as
``ops.PagedKV``, ``ops.paged_attention`` and so on.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from ._native import DA_F32, PagedBatchBlock, PagedKVBlock, call_on, check, dtype_code, lib
from .kv4 import _gpu

__all__ = ["PagedKV", "PagedBatch", "append_paged", "paged_attention", "shared_prefix_attention"]

_I32, _U8 = torch.int32, torch.uint8


class PagedKV:
    """The pages of one layer: ``k_pages``, ``v_pages`` [num_pages, Hkv, page_size, D] of one type
    (bf16, fp16 or fp32).  Any strides that are multiples of 8 elements with a contiguous head
    dimension (a view of [num_pages, page_size, Hkv, D] too); ``page_size`` a power of two from 16
    on, D a multiple of 8 up to 128.  The tensors of an object are fixed, their contents are not."""

    __slots__ = ("k_pages", "v_pages", "num_pages", "kv_heads", "page_size", "head_dim", "dtype", "device", "_index",
                 "_code", "_block", "_ref")

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor):
        shape, device, index = k_pages.shape, _gpu(k_pages, "k_pages"), k_pages.get_device()
        if len(shape) != 4 or v_pages.shape != shape or v_pages.get_device() != index:
            raise ValueError("k_pages and v_pages are [num_pages, Hkv, page_size, D] of one shape on one device")
        code = dtype_code(k_pages, v_pages)
        P, H, S, D = shape
        if not (P and H):
            raise ValueError("a cache needs pages and heads")
        if S < 16 or S & (S - 1):
            raise ValueError(f"page_size must be a power of two from 16 on, got {S}")
        if D <= 0 or D > 128 or D % 8:
            raise ValueError(f"head_dim must be a multiple of 8 in [8, 128], got {D}")
        sk, sv = k_pages.stride(), v_pages.stride()
        kp, vp = k_pages.data_ptr(), v_pages.data_ptr()
        if sk[3] != 1 or sv[3] != 1 or (sk[0] | sk[1] | sk[2] | sv[0] | sv[1] | sv[2]) % 8 or (kp | vp) % 16:
            raise ValueError("pages need a contiguous head dimension, strides that are multiples of 8 elements and "
                             "16-byte alignment")
        self.k_pages, self.v_pages = k_pages, v_pages
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = P, H, S, D
        self.dtype, self.device, self._index, self._code = k_pages.dtype, device, index, code
        self._block = PagedKVBlock(kp, vp, P, S, sk[0], sk[1], sk[2], sv[0], sv[1], sv[2])
        self._ref = ctypes.byref(self._block)


def _ints(t: torch.Tensor, name: str, n: int, index: int) -> int:
    """The address of an int32 tensor of n values on GPU ``index``."""
    if t.dtype is not _I32 or t.shape != (n,) or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} values on cuda:{index}")
    return t.data_ptr()


class PagedBatch:
    """The sequences of a call, on the device.

    ``table`` [B, width] int32 names each sequence's pages in order (entries past them may hold
    anything), ``lengths`` [B] int32 its tokens in them, those that the call brings included, and last.
    ``cu_seqlens`` [B + 1] int32: sequence b brings tokens cu[b] .. cu[b + 1] - 1 of q, k, v [T, heads, D],
    at most ``max_seqlen``; without it every sequence brings one (token b).  Tokens past cu[B] are left
    alone, so a batch may be padded.  ``start`` [B] int32: the position of a sequence's first token in
    its pages (default 0; a sequence behind a shared prefix starts at the prefix's length).  A list or
    a CPU tensor of cu_seqlens is checked, copied to the device and gives ``max_seqlen``.  The tensors
    are fixed, their contents are not."""

    __slots__ = ("table", "lengths", "cu", "start", "batch", "max_seqlen", "device", "_index", "_block", "_ref")

    def __init__(self, table: torch.Tensor, lengths: torch.Tensor, cu_seqlens=None, max_seqlen: Optional[int] = None,
                 start: Optional[torch.Tensor] = None):
        device, index = _gpu(table, "table"), table.get_device()
        shape, stride = table.shape, table.stride()
        if len(shape) != 2 or stride[1] != 1 or table.dtype is not _I32 or 0 in shape:
            raise ValueError("table must be int32 [B, width] with contiguous rows")
        B, width = shape
        cu = cu_seqlens
        if cu is not None and not (isinstance(cu, torch.Tensor) and cu.device.type == "cuda"):
            host = [int(x) for x in (cu.tolist() if isinstance(cu, torch.Tensor) else cu)]
            if len(host) != B + 1 or host[0] != 0 or any(y < x for x, y in zip(host, host[1:])):
                raise ValueError(f"cu_seqlens must rise from 0 over {B} sequences, got {host}")
            longest = max(1, max(y - x for x, y in zip(host, host[1:])))
            max_seqlen = longest if max_seqlen is None else max(longest, int(max_seqlen))
            cu = torch.tensor(host, dtype=_I32, device=device)
        if cu is None:
            at_cu, max_seqlen = None, 1
        else:
            at_cu = _ints(cu, "cu_seqlens", B + 1, index)
            if max_seqlen is None or max_seqlen <= 0:
                raise ValueError("max_seqlen (the most tokens a sequence brings) is needed with cu_seqlens on the device")
        self.table, self.lengths, self.cu, self.start = table, lengths, cu, start
        self.batch, self.max_seqlen, self.device, self._index = B, int(max_seqlen), device, index
        self._block = PagedBatchBlock(table.data_ptr(), _ints(lengths, "lengths", B, index), at_cu,
                                      None if start is None else _ints(start, "start", B, index), B, width, stride[0],
                                      self.max_seqlen)
        self._ref = ctypes.byref(self._block)


def _tokens(t: torch.Tensor, name: str, kv: PagedKV):
    """(t, its shape, its strides) of a [T, heads, D] tensor that fits the pages; a copy where its rows do
    not begin at multiples of 16 bytes."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != kv.head_dim or t.dtype is not kv.dtype or t.get_device() != kv._index:
        raise ValueError(f"{name} must be [tokens, heads, {kv.head_dim}] {kv.dtype} on {kv.device}, got "
                         f"{list(shape)} {t.dtype} on {t.device}")
    s = t.stride()
    if s[2] != 1 or (s[0] | s[1]) & 7 or t.data_ptr() & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        s = t.stride()
    return t, shape, s


def _output(out: Optional[torch.Tensor], q: torch.Tensor, shape, name: str) -> torch.Tensor:
    if out is None:
        return q.new_empty(shape)
    if out.shape != shape or out.dtype is not q.dtype or out.get_device() != q.get_device() or out.stride(2) != 1 or out.data_ptr() & 15:
        raise ValueError(f"{name} must have q's shape, type and device, a contiguous head dimension and 16-byte alignment")
    return out


def _batch(batch: PagedBatch, kv: PagedKV, T: int) -> None:
    if batch._index != kv._index:
        raise ValueError(f"the batch is on {batch.device}, the pages on {kv.device}")
    if batch.cu is None and batch.batch > T:
        raise ValueError(f"{T} tokens for {batch.batch} sequences of one each")


def append_paged(kv: PagedKV, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor, q: Optional[torch.Tensor] = None,
                 cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, interleaved: bool = False,
                 per_token: bool = False, out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """New tokens k, v [T, Hkv, D] into the pages of ``batch``, the keys rotated to their positions; the
    queries q [T, Hq, D], rotated too, are returned (in ``out``, which may be q).

    cos, sin [rows, R / 2] (float32 or the pages' type, contiguous along R / 2; R a multiple of 4 up to
    D): row p is for position p, with ``per_token`` row t for token t.  Dims d and d + R / 2 (with
    ``interleaved`` 2 d and 2 d + 1) are a pair, turned in float32 and rounded once; dims from R on
    stay.  A position outside the rows takes the nearest one.  Without cos and sin nothing is rotated.
    Tokens past the batch's last are left alone, and a token whose place is not in the table is not written
    (its query is rotated); two tokens meant for one place leave either of them there.
    """
    k, shape, sk = _tokens(k, "k", kv)
    v, of_v, sv = _tokens(v, "v", kv)
    T, H, D = shape
    if H != kv.kv_heads or of_v != shape or not T:
        raise ValueError(f"k and v must be [tokens, {kv.kv_heads}, {D}], got {list(shape)} and {list(of_v)}")
    _batch(batch, kv, T)
    sq, so, Hq, qp, op = (0, 0), (0, 0), 0, None, None
    if q is not None:
        src, of_q, sq = _tokens(q, "q", kv)
        Hq = of_q[1]
        if of_q[0] != T or not Hq:
            raise ValueError(f"q {list(of_q)} must hold the {T} tokens of k")
        out = _output(out, q, of_q, "out")
        so, qp, op = out.stride(), src.data_ptr(), out.data_ptr()
    elif out is not None:
        raise ValueError("out is for the rotated queries: it needs q")
    rows = s_rot = rot = 0
    code, cp, sp = kv._code, None, None
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        table, s = cos.shape, cos.stride()
        if len(table) != 2 or sin.shape != table or sin.dtype is not cos.dtype or cos.get_device() != kv._index \
                or sin.get_device() != kv._index or s[1] != 1 or sin.stride() != s:
            raise ValueError("cos and sin must be [rows, R / 2] of one shape, type and stride on the pages' device")
        rows, rot, s_rot = table[0], 2 * table[1], s[0]
        if cos.dtype is torch.float32:
            code = DA_F32
        elif cos.dtype is not kv.dtype:
            raise TypeError(f"cos and sin must be torch.float32 or {kv.dtype}, got {cos.dtype}")
        if not rows or not rot or rot % 4 or rot > D:
            raise ValueError(f"cos and sin of {list(table)} do not fit a head_dim of {D}: R is a multiple of 4")
        if per_token and rows < T:
            raise ValueError(f"{rows} rows of cos and sin for {T} tokens")
        cp, sp = cos.data_ptr(), sin.data_ptr()
    rc = call_on(kv.device, lib().da_paged_append, k.data_ptr(), sk[0], sk[1], v.data_ptr(), sv[0], sv[1], qp, sq[0], sq[1],
                 op, so[0], so[1], kv._code, T, Hq, H, D, cp, sp, code, rows, s_rot, rot, 1 if interleaved else 0,
                 1 if per_token else 0, kv._ref, batch._ref)
    check(rc, "da_paged_append")
    return out


def _attention(q, kv, batch, prefix, scale, out):
    src, shape, sq = _tokens(q, "q", kv)
    T, Hq, D = shape
    H = kv.kv_heads
    if not T or not Hq or Hq % H:
        raise ValueError(f"{T} tokens of {Hq} query heads over {H} KV heads")
    _batch(batch, kv, T)
    out = _output(out, q, shape, "out")
    so = out.stride()
    common = None if prefix is None else prefix._ref
    native = lib()
    n = native.da_paged_attention_workspace_size(kv._code, T, Hq, H, D, kv._ref, batch._ref, common)
    ws = torch.empty((n,), dtype=_U8, device=kv.device) if n > 0 else None  # held until the call is on its stream
    rc = call_on(kv.device, native.da_paged_attention, src.data_ptr(), sq[0], sq[1], out.data_ptr(), so[0], so[1], kv._code,
                 T, Hq, H, D, D ** -0.5 if scale is None else scale, kv._ref, batch._ref, common,
                 None if ws is None else ws.data_ptr(), n)
    check(rc, "da_paged_attention")
    return out


def paged_attention(q: torch.Tensor, kv: PagedKV, batch: PagedBatch, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of the new tokens q [T, Hq, D] (already rotated, their keys and values already
    in the pages): query token i of the n that sequence b brings sees the keys of slots 0 ..
    lengths[b] - n + i.  One token a sequence is a decode step; many are a prompt, or the next part of one;
    both may come in one batch.  Query head h reads KV head h // (Hq // Hkv).  A query without any key
    gives zeros; rows of tokens past the batch's last, or past a sequence's ``max_seqlen``, are left as
    ``out`` has them."""
    return _attention(q, kv, batch, None, scale, out)


def shared_prefix_attention(q: torch.Tensor, kv: PagedKV, batch: PagedBatch, prefix: PagedBatch,
                            scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``paged_attention`` where groups of sequences have their first tokens in common: ``prefix``
    holds a row of ``table`` and ``lengths`` for every group, and ``cu_seqlens`` over q's tokens
    says which are the group's (whole sequences, in order; ``max_seqlen`` the most tokens of a group).
    Every query of a group sees all of its prefix and then its own sequence as in ``paged_attention``;
    tokens past the group's ``max_seqlen`` are left as ``out`` has them.
    The prefix's keys and values are read once for the group, not once for each sequence."""
    if prefix.cu is None:
        raise ValueError("prefix needs cu_seqlens: which of q's tokens belong to which group")
    if prefix._index != kv._index:
        raise ValueError(f"the prefix is on {prefix.device}, the pages on {kv.device}")
    return _attention(q, kv, batch, prefix, scale, out)
