"""A PagedCache on the CPU, its kernels replaced by torch indexing: what the cache itself does, without a
GPU.  Test infrastructure."""
import types

import pytest
import torch

from deltaattention_amd import paged_cache


class Kernels:
    """Stands for ``deltaattention_amd.paged``.  ``fail``: the next append raises it."""

    def __init__(self):
        self.fail = None

    @staticmethod
    def PagedKV(k, v):
        return k, v

    @staticmethod
    def PagedBatch(table, lengths, cu=None, max_seqlen=None, start=None):
        return types.SimpleNamespace(table=table, lengths=lengths, max_seqlen=max_seqlen)

    def append_paged(self, kv, batch, k, v, q=None, cos=None, sin=None, per_token=False):
        if self.fail is not None:
            fail, self.fail = self.fail, None
            raise fail
        if cos is not None and (cos.shape != sin.shape or cos.dtype != sin.dtype or cos.stride() != sin.stride()):
            raise ValueError("cos and sin must be of one shape, type and stride")
        B, page = batch.table.shape[0], kv[0].shape[2]
        n = k.shape[0] // B
        for b in range(B):
            for i in range(n):
                slot = int(batch.lengths[b]) - n + i
                at = int(batch.table[b, slot // page])
                kv[0][at, :, slot % page], kv[1][at, :, slot % page] = k[b * n + i], v[b * n + i]
        return q

    @staticmethod
    def paged_attention(q, kv, batch, scale=None):
        return q

    @staticmethod
    def shared_prefix_attention(q, kv, batch, prefix, scale=None):
        return q


@pytest.fixture
def kernels(monkeypatch):
    made = Kernels()
    monkeypatch.setattr(paged_cache, "paged", made)
    return made


def config(layers=1, heads=4, kv=2, dim=16):
    return types.SimpleNamespace(head_dim=dim, num_key_value_heads=kv, num_hidden_layers=layers, hidden_size=heads * dim,
                                 num_attention_heads=heads)


def cache(batch=2, layers=1, pages=60, dtype=torch.float32):
    return paged_cache.PagedCache(config(layers), batch, dtype=dtype, num_pages=pages, device="cpu")


def tokens(batch, n, heads=2, seed=0, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(batch, heads, n, 16, generator=gen).to(dtype) for _ in range(2)]


def held(c, layer=0):
    """The cache's own keys and values [B, H, tokens, D], gathered from its pages."""
    table = c._table[:, :len(c._pages[0])].long()
    return [p[layer][table].transpose(1, 2).reshape(c.bsz, p.shape[2], -1, p.shape[4])[:, :, :c._seen[layer]]
            for p in (c._pool.k, c._pool.v)]


def state(c):
    return (c._total, list(c._seen), [list(p) for p in c._pages], sorted(c._pool.free), list(c._pool.holders),
            c._lengths.tolist(), c._batch, c._prefix)
