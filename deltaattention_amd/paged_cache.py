"""``PagedCache``: the exact key/value cache of the model swap, in pages.

The reference's dense path keeps no cache of its own (modeling_llama.py:778-803) and its compressed
cache replaces most tokens by anchors.  This one holds every token at full width, continues a
sequence with one token or many, and lets several sequences share a prompt (``fork``), whose pages are
then stored once and read once a step.  Built on ``ops.append_paged``, ``ops.paged_attention`` and
``ops.shared_prefix_attention``; ``llama_swap.install`` routes a model through it.
"""
from __future__ import annotations

from typing import List, Optional

import torch

from . import paged
from ._native import _raw_stream

try:
    from transformers import Cache as _CacheBase
except Exception:  # pragma: no cover - transformers is optional for the kernels
    _CacheBase = object

__all__ = ["PagedCache"]


def _indexed(device) -> torch.device:
    """``device`` with its index: "cuda" is the device that is current now, whichever is later."""
    device = torch.device(device)
    return torch.device("cuda", torch.cuda.current_device()) if device.type == "cuda" and device.index is None else device


def _stream_of(index: Optional[int]) -> int:
    """The handle of the current stream of GPU ``index`` (None: the CPU)."""
    return 0 if index is None else _raw_stream(index)


def _keep(tensors, stream) -> None:
    """Their memory stays until what ``stream`` has been given by the time they go is done."""
    for t in tensors:
        if t is not None:
            t.record_stream(stream)


class _Pool:
    """Pages of every layer, k and v [L, pages, Hkv, page_size, D], how many hold each page, and which
    are free.  A cache and its forks have one pool, whose work is in one order whichever streams they are used
    from: a page that one gives back, or memory that one's growth replaces, is another's in the same call."""

    def __init__(self, layers, pages, heads, page_size, head_dim, dtype, device):
        shape = (layers, pages, heads, page_size, head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty_like(self.k)
        self.holders = [0] * pages
        self.free = list(range(pages - 1, -1, -1))
        self._views()
        self.device, self.index = self.k.device, self.k.device.index
        self.raw = _stream_of(self.index)           # the stream that was used last
        self.stream = torch.cuda.current_stream(self.device) if self.k.is_cuda else None

    def enter(self) -> None:
        """The current stream goes on after all that the pool's caches have queued on another one.  (Not within a
        capture, which may not wait for work outside of it, and begins with a synchronization.)"""
        raw = _stream_of(self.index)
        if raw == self.raw or torch.cuda.is_current_stream_capturing():
            return
        now = torch.cuda.current_stream(self.device)
        now.wait_stream(self.stream)
        _keep((self.k, self.v), now)
        self.raw, self.stream = raw, now

    def _views(self):
        n = len(self.holders)
        self.layers = [paged.PagedKV(k[:n], v[:n]) for k, v in zip(self.k, self.v)]

    def grow(self, pages):
        """To ``pages`` pages, contents kept.  Where memory for v is short after k has its own, k stays the larger
        one and all else as it was."""
        old = len(self.holders)
        for name in ("k", "v"):
            t = getattr(self, name)
            if t.shape[1] >= pages:
                continue
            new = torch.empty((t.shape[0], pages, *t.shape[2:]), dtype=t.dtype, device=t.device)
            new[:, :old] = t[:, :old]
            setattr(self, name, new)
            self._views()
        self.holders += [0] * (pages - old)
        self.free = list(range(pages - 1, old - 1, -1)) + self.free
        self._views()

    def take(self, n) -> List[int]:
        if n > len(self.free):
            self.grow(max(2 * len(self.holders), len(self.holders) + n))
        out = [self.free.pop() for _ in range(n)]
        for p in out:
            self.holders[p] = 1
        return out

    def hold(self, pages):
        for p in pages:
            self.holders[p] += 1

    def drop(self, pages):
        for p in pages:
            self.holders[p] -= 1
            if self.holders[p] == 0:
                self.free.append(p)


class PagedCache(_CacheBase):
    """An exact cache of ``batch_size`` sequences of equal length (no padding) in pages of ``page_size``
    tokens.  ``num_pages`` (default: 1024 tokens a sequence) is a first size: the pool grows.

    Every layer has the same tokens in the same pages.  A step brings n tokens a sequence to each layer in
    turn: ``append`` (keys rotated on the way) then ``attend``.  A call that is refused changes nothing.
    A step's batch lies in tensors that the next step changes in place.  Calls may come from different
    streams: those of a cache and of its forks, which share its pages, run in the order in which they
    were made.  They have to come from one thread at a time.
    """

    def __init__(self, config, batch_size, dtype=torch.bfloat16, page_size: int = 16, num_pages: Optional[int] = None,
                 device="cuda", _of: Optional["PagedCache"] = None, _copies: int = 1):
        if _CacheBase is not object:
            try:
                super().__init__(layers=[])
            except TypeError:
                super().__init__()
        self.bsz, self.dtype, self.device = int(batch_size), dtype, _indexed(device)
        if self.bsz <= 0 or page_size <= 0:
            raise ValueError(f"{batch_size} sequences, pages of {page_size} tokens")
        self.prefix_length, self._copies, self._common = 0, _copies, None
        if _of is None:
            self.head_dim = getattr(config, "head_dim", None) or config.hidden_size // config.num_attention_heads
            self.n_kv_heads = config.num_key_value_heads
            self.num_layers, self.page_size = config.num_hidden_layers, int(page_size)
            pages = self.bsz * -(-1024 // self.page_size) if num_pages is None else int(num_pages)
            self._pool = _Pool(self.num_layers, max(1, pages), self.n_kv_heads, self.page_size, self.head_dim, dtype,
                               self.device)
        else:
            _of._enter()
            for name in ("head_dim", "n_kv_heads", "num_layers", "page_size", "_pool"):
                setattr(self, name, getattr(_of, name))
            self.prefix_length = _of._total
            self._common = [list(p) for p in _of._pages]
            for p in self._common:
                self._pool.hold(p)
            self._prefix_table = _of._table.clone()
            self._prefix_lengths = _of._lengths.clone()
        self._pages: List[List[int]] = [[] for _ in range(self.bsz)]
        self._table = torch.zeros((self.bsz, 1), dtype=torch.int32, device=self.device)
        self._lengths = torch.zeros((self.bsz,), dtype=torch.int32, device=self.device)
        self._start = None if not self.prefix_length else torch.full_like(self._lengths, self.prefix_length)
        self._total = 0                             # own tokens of a sequence, the step in progress included
        self._seen = [0] * self.num_layers          # those of each layer
        self._batch = self._prefix = None           # of the step in progress
        self._cu = {}
        self._raw = self._pool.raw                  # the stream that was used last

    # ---- pages ----

    def _enter(self) -> None:
        """Before every use of the pages and of the cache's own tensors on the current stream."""
        pool = self._pool
        if _stream_of(pool.index) != pool.raw:
            pool.enter()
        if self._raw != pool.raw:
            more = () if self._common is None else (self._prefix_table, self._prefix_lengths)
            _keep((self._table, self._lengths, self._start, *more, *self._cu.values()), pool.stream)
            self._raw = pool.raw

    def _starts(self, rows: int, n: int) -> torch.Tensor:
        """0, n, 2 n, .. for ``rows`` entries."""
        key = rows, n
        if key not in self._cu:
            if len(self._cu) > 64:
                self._cu.clear()
            self._cu[key] = torch.arange(0, rows * n + 1, n, dtype=torch.int32, device=self.device)
        return self._cu[key]

    def _begin(self, layer_idx: int, n: int) -> None:
        """Room for n tokens of this layer: made by the first layer of a step, there for the others."""
        want = self._seen[layer_idx] + n
        if want == self._total and self._batch is not None:
            return
        if any(x != self._total for x in self._seen):
            raise RuntimeError(f"layer {layer_idx} brings {n} tokens to {self._seen[layer_idx]}, but the layers of one step "
                               f"have to bring the same ({self._total} in all)")
        have = len(self._pages[0])
        more = -(-want // self.page_size) - have
        if more > 0:
            taken = self._pool.take(more * self.bsz)
            rows = [taken[b * more:(b + 1) * more] for b in range(self.bsz)]
            for mine, new in zip(self._pages, rows):
                mine.extend(new)
            if have + more > self._table.shape[1]:
                wide = torch.zeros((self.bsz, max(2 * self._table.shape[1], have + more)), dtype=torch.int32, device=self.device)
                wide[:, :have] = self._table[:, :have]
                self._table = wide
            self._table[:, have:have + more] = torch.tensor(rows, dtype=torch.int32).to(self.device)
        self._lengths.fill_(want)
        self._total = want
        cu = None if n == 1 else self._starts(self.bsz, n)
        # of the table only the columns in use: what the kernels plan with
        self._batch = paged.PagedBatch(self._table[:, :len(self._pages[0])], self._lengths, cu, n, start=self._start)
        if self._common is not None:
            group = self._copies * n
            self._prefix = paged.PagedBatch(self._prefix_table, self._prefix_lengths,
                                            self._starts(self.bsz // self._copies, group), group)

    def _step(self):
        """What a step changes before its first kernel runs, for ``_back``."""
        return self._total, self._batch, self._prefix, len(self._pages[0])

    def _back(self, step) -> None:
        """To what ``_step`` gave: the pages taken since go back, the lengths on the device are those before."""
        self._total, self._batch, self._prefix, have = step
        for mine in self._pages:
            self._pool.drop(mine[have:])
            del mine[have:]
        self._lengths.fill_(self._total)

    def fork(self, copies: int) -> "PagedCache":
        """A cache of ``copies`` sequences for each one here, in order, all behind this cache's tokens as
        they are now: these pages are not copied, and read once for the copies of a sequence.  This cache may
        go on by itself."""
        if self._common is not None:
            raise NotImplementedError("a forked cache cannot be forked again")
        if copies <= 0 or not self._total or any(x != self._total for x in self._seen):
            raise ValueError(f"fork({copies}) of {self._total} tokens, {self._seen} of them in the layers")
        return PagedCache(None, self.bsz * copies, self.dtype, self.page_size, device=self.device, _of=self, _copies=copies)

    def reset(self) -> None:
        """Empties the cache and gives its pages back (those of a shared prefix stay)."""
        for p in self._pages:
            self._pool.drop(p)
        self._pages = [[] for _ in range(self.bsz)]
        self._total, self._seen, self._batch, self._prefix = 0, [0] * self.num_layers, None, None

    def __del__(self):
        pool = getattr(self, "_pool", None)
        if pool is not None:
            for p in getattr(self, "_pages", []) + (getattr(self, "_common", None) or []):
                pool.drop(p)

    # ---- a step ----

    def _tokens(self, t: torch.Tensor, name: str, heads: Optional[int] = None) -> torch.Tensor:
        """[B, heads, N, D] as [B * N, heads, D]."""
        if t.dim() != 4 or t.shape[0] != self.bsz or t.shape[3] != self.head_dim or not t.shape[2] \
                or (heads is not None and t.shape[1] != heads) or t.shape[1] % self.n_kv_heads:
            raise ValueError(f"{name} must be [{self.bsz}, heads, tokens, {self.head_dim}] over {self.n_kv_heads} KV heads, got "
                             f"{list(t.shape)}")
        if t.dtype != self.dtype or t.device != self._lengths.device:
            raise ValueError(f"{name} is {t.dtype} on {t.device}, the cache {self.dtype} on {self._lengths.device}")
        return t.transpose(1, 2).reshape(-1, t.shape[1], self.head_dim)

    def append(self, key: torch.Tensor, value: torch.Tensor, layer_idx: int, query: Optional[torch.Tensor] = None,
               cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """A step's key, value [B, Hkv, N, D] into the layer's pages.  With cos and sin [B or 1, N, R] (a model's
        position embeddings, whose two halves are alike: the first is read) keys, and query [B, Hq, N, D], are
        rotated.  Returns the query as [B * N, Hq, D], rotated or as it was."""
        k, v = self._tokens(key, "key", self.n_kv_heads), self._tokens(value, "value", self.n_kv_heads)
        n = key.shape[2]
        if value.shape[2] != n or (query is not None and query.shape[2] != n):
            raise ValueError(f"key, value and query bring {n}, {value.shape[2]} and "
                             f"{None if query is None else query.shape[2]} tokens")
        q = None if query is None else self._tokens(query, "query")
        if (cos is None) != (sin is None):
            raise ValueError("cos and sin come together")
        if cos is not None:
            cos, sin = self._rows(cos, n), self._rows(sin, n)
            if cos.stride() != sin.stride():
                cos, sin = cos.contiguous(), sin.contiguous()
        self._enter()
        before = self._step()
        try:
            self._begin(layer_idx, n)
            got = paged.append_paged(self._pool.layers[layer_idx], self._batch, k, v, q=None if cos is None else q, cos=cos,
                                     sin=sin, per_token=True)
        except BaseException:
            if before != self._step():
                self._back(before)
            raise
        self._seen[layer_idx] += n
        return q if cos is None else got

    def _rows(self, t: torch.Tensor, n: int) -> torch.Tensor:
        """Position embeddings [B or 1, N, R] as a row of R / 2 a token."""
        if t.dim() != 3 or t.shape[0] not in (1, self.bsz) or t.shape[1] != n or t.shape[2] > self.head_dim or t.shape[2] % 8 \
                or t.device != self._lengths.device or t.dtype not in (torch.float32, self.dtype):
            raise ValueError(f"cos and sin must be [{self.bsz} or 1, {n}, R] in float32 or {self.dtype}, got {list(t.shape)} "
                             f"{t.dtype} on {t.device}")
        if t.shape[0] != self.bsz:
            t = t.expand(self.bsz, -1, -1)
        return t.reshape(-1, t.shape[2])[:, :t.shape[2] // 2]

    def attend(self, query: torch.Tensor, layer_idx: int, scaling: Optional[float] = None) -> torch.Tensor:
        """The step's queries [B * N, Hq, D] (as ``append`` returns them) over the layer: [B, N, Hq, D]."""
        if self._batch is None or self._seen[layer_idx] != self._total:
            raise RuntimeError("attend follows the append of the same step and layer")
        n = self._batch.max_seqlen
        if query.dim() != 3 or query.shape[0] != self.bsz * n:
            raise ValueError(f"query must hold the step's {n} tokens of {self.bsz} sequences, got {list(query.shape)}")
        self._enter()
        kv = self._pool.layers[layer_idx]
        if self._prefix is None:
            out = paged.paged_attention(query, kv, self._batch, scale=scaling)
        else:
            out = paged.shared_prefix_attention(query, kv, self._batch, self._prefix, scale=scaling)
        return out.view(self.bsz, -1, *out.shape[1:])

    # ---- transformers' cache interface ----

    def get_seq_length(self, layer_idx: int = 0) -> int:
        return self.prefix_length + self._seen[layer_idx]

    def get_max_length(self):
        return None

    def get_max_cache_shape(self, layer_idx: int = 0):
        return None

    def update(self, key_states, value_states, layer_idx, cache_kwargs=None):
        raise NotImplementedError("a PagedCache does not give its keys back: llama_swap.install(model) runs the attention "
                                  "over its pages")

    def crop(self, max_length: int) -> None:
        raise NotImplementedError("a PagedCache is not cropped")

    def reorder_cache(self, beam_idx) -> None:
        raise NotImplementedError("the sequences of a PagedCache keep their order")

    def batch_repeat_interleave(self, repeats: int) -> None:
        raise NotImplementedError("PagedCache.fork(copies) gives a cache of several sequences behind one prompt")

    def batch_select_indices(self, indices) -> None:
        raise NotImplementedError("the sequences of a PagedCache keep their order")
