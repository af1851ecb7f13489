"""A PagedCache and its forks used from several streams: their work is in one order, and memory stays until all
streams that use it are done with it."""
import types

import pytest
import torch

from conftest import announce
from paged_cache_on_cpu import cache, kernels, tokens  # noqa: F401 (kernels: a fixture)


class Stream:
    def __init__(self, raw, log):
        self.raw, self.log = raw, log

    def wait_stream(self, other):
        self.log.append((self.raw, "after", other.raw))


@pytest.fixture
def streams(monkeypatch):
    """Streams by number, on the CPU: the one that is current, and what was asked of them."""
    from deltaattention_amd import paged_cache
    at = types.SimpleNamespace(now=1, log=[], kept=[], capturing=False)
    made = {}
    current = lambda *a: made.setdefault(at.now, Stream(at.now, at.log))  # noqa: E731
    monkeypatch.setattr(paged_cache, "_stream_of", lambda device: at.now, raising=False)
    monkeypatch.setattr(paged_cache, "_keep", lambda tensors, s: at.kept.extend((t, s.raw) for t in tensors if t is not None),
                        raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", current)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: at.capturing)
    at.current = current
    return at


def _made(streams):
    c = cache()
    c._pool.stream = streams.current()  # of a CPU pool there is none
    return c


def test_calls_wait_for_the_stream_before(kernels, streams):  # noqa: F811
    c = _made(streams)
    c.append(*tokens(2, 20), 0)
    assert streams.log == []
    streams.now = 2
    fork = c.fork(2)
    assert streams.log == [(2, "after", 1)]
    fork.append(*tokens(4, 3), 0)
    streams.now = 1
    q = c.append(*tokens(2, 1), 0, tokens(2, 1, 4)[0])
    assert streams.log[1:] == [(1, "after", 2)]
    streams.now = 3
    c.attend(q, 0)
    assert streams.log[2:] == [(3, "after", 1)]
    c.attend(q, 0)
    assert len(streams.log) == 3
    streams.now, streams.capturing = 4, True
    c.attend(q, 0)
    assert len(streams.log) == 3


def test_memory_is_kept_for_every_stream(kernels, streams):  # noqa: F811
    c = _made(streams)
    c.append(*tokens(2, 3), 0)
    q = tokens(2, 3, 4)[0]
    fork = c.fork(1)
    streams.now = 2
    fork.append(*tokens(2, 3), 0, q)
    mine = lambda c: [c._table, c._lengths, *c._cu.values()]  # noqa: E731
    kept = {(t.data_ptr(), s) for t, s in streams.kept}
    for t in [c._pool.k, c._pool.v, fork._prefix_table, fork._prefix_lengths, fork._start, fork._table, fork._lengths]:
        assert (t.data_ptr(), 2) in kept
    assert not any((t.data_ptr(), 2) in kept for t in mine(c))
    c.append(*tokens(2, 3), 0, q)  # the pool was last used on this stream, this cache was not
    kept = {(t.data_ptr(), s) for t, s in streams.kept}
    assert all((t.data_ptr(), 2) in kept for t in mine(c))


def _twins(config):
    from deltaattention_amd.paged_cache import PagedCache
    return [PagedCache(config, 2, num_pages=6) for _ in range(2)]


@pytest.mark.gpu
def test_parent_and_fork_on_two_streams(gpu):
    """The parent's and the fork's steps, the pool's growth and pages that come back, with one stream held up by
    other work each time the other one is used, against the same calls on one stream."""
    announce("PagedCache: parent and fork on two streams")
    config = types.SimpleNamespace(head_dim=64, num_key_value_heads=2, num_hidden_layers=2, hidden_size=256,
                                   num_attention_heads=4)
    gen = torch.Generator().manual_seed(3)
    data = {}

    def given(name, B, n):
        if name not in data:
            data[name] = [torch.randn(B, h, n, 64, generator=gen).bfloat16().to(gpu) for h in (4, 2, 2)]
        return data[name]
    busy = torch.randn(4096, 4096, device=gpu).bfloat16()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    one, two = _twins(config)
    results = []
    for parent, streams in ((one, None), (two, (a, b))):
        torch.cuda.synchronize()
        out = []

        def step(cache, name, B, n, which):
            q, k, v = given(name, B, n)

            def run():
                for layer in range(2):
                    out.append(cache.attend(cache.append(k, v, layer, q), layer))
            if streams is None:
                return run()
            with torch.cuda.stream(streams[which]):
                hold = busy
                for _ in range(10):
                    hold = hold @ busy
                run()
        for name, B, n in (("p0", 2, 30), ("f0", 6, 5), ("p1", 2, 100), ("f1", 6, 60), ("p2", 2, 1), ("f2", 6, 1), ("p3", 2, 70),
                           ("g0", 4, 20)):
            given(name, B, n)
        torch.cuda.synchronize()
        step(parent, "p0", 2, 30, 0)
        fork = parent.fork(3)
        step(fork, "f0", 6, 5, 1)
        step(parent, "p1", 2, 100, 0)   # grows the pool
        step(fork, "f1", 6, 60, 1)      # grows it again
        step(parent, "p2", 2, 1, 0)
        step(fork, "f2", 6, 1, 1)
        fork.reset()                    # its pages go to the next one, on the other stream
        step(parent, "p3", 2, 70, 0)
        other = parent.fork(2)
        del fork
        step(other, "g0", 4, 20, 1)
        torch.cuda.synchronize()
        results.append(out)
    for got, want in zip(*results):
        assert torch.isfinite(want).all() and torch.equal(got, want)
