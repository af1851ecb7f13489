"""A PagedCache's pool that runs out of memory while it grows (on the CPU, kernels replaced)."""
import pytest
import torch

from paged_cache_on_cpu import cache, held, kernels, state, tokens  # noqa: F401 (kernels: a fixture)


def _without_memory(monkeypatch, after):
    """torch.empty fails for a pool's tensors after so many of them."""
    real, left = torch.empty, [after]

    def empty(shape, *args, **more):
        if isinstance(shape, tuple) and len(shape) == 5:
            left[0] -= 1
            if left[0] < 0:
                raise torch.OutOfMemoryError("no memory")
        return real(shape, *args, **more)
    monkeypatch.setattr(torch, "empty", empty)


@pytest.mark.parametrize("pages", [4, 7])
@pytest.mark.parametrize("after", [0, 1])
def test_growth_without_memory(kernels, monkeypatch, after, pages):  # noqa: F811
    """k or v cannot be had: what is held stays, writes go on, and a later growth has all of it."""
    c = cache(layers=2, pages=pages)
    first = tokens(2, 20)
    for layer in range(2):
        c.append(*first, layer)
    before = state(c)
    for _ in range(2):
        with monkeypatch.context() as m:
            _without_memory(m, after)
            with pytest.raises(torch.OutOfMemoryError):
                c.append(*tokens(2, 90, seed=1), 0)
            after = 0 if after else after  # the larger k is there already
        assert state(c) == before
    more = [tokens(2, n, seed=n) for n in (3, 9, 90, 300)]  # within the pages that are there, then beyond
    for t in more:
        for layer in range(2):
            c.append(*t, layer)
    for layer in range(2):
        for i, got in enumerate(held(c, layer)):
            assert torch.equal(got, torch.cat([first[i]] + [t[i] for t in more], 2))
    assert c._pool.k.shape == c._pool.v.shape and c._pool.k.shape[1] == len(c._pool.holders)
    assert sum(x > 0 for x in c._pool.holders) == 2 * len(c._pages[0]) == len(c._pool.holders) - len(c._pool.free)
