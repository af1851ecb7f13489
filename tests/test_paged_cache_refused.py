"""A PagedCache's calls that are refused, or that fail, change nothing (on the CPU, kernels replaced)."""
import pytest
import torch

from paged_cache_on_cpu import cache, held, kernels, state, tokens  # noqa: F401 (kernels: a fixture)


def _begun(layers=1, dtype=torch.float32):
    """A cache of 20 tokens and what it holds."""
    c = cache(layers=layers, dtype=dtype)
    k, v = tokens(2, 20, dtype=dtype)
    for layer in range(layers):
        c.append(k, v, layer)
    return c, (k, v)


@pytest.mark.parametrize("what", ["width", "type", "sin alone", "cos alone"])
def test_cos_and_sin_that_differ(kernels, what):  # noqa: F811
    low = torch.bfloat16
    c, first = _begun(dtype=low)
    k, v = tokens(2, 30, seed=1, dtype=low)
    cos = torch.ones(1, 30, 16)
    cos, sin = {"width": (cos, torch.ones(1, 30, 8)), "type": (cos, cos.to(low)), "sin alone": (None, cos),
                "cos alone": (cos, None)}[what]
    before = state(c)
    with pytest.raises((ValueError, TypeError)):
        c.append(k, v, 0, tokens(2, 30, 4, dtype=low)[0], cos, sin)
    assert state(c) == before
    more = tokens(2, 7, seed=2, dtype=low)
    c.append(*more, 0)  # the cache goes on, with another number of tokens
    for got, a, b in zip(held(c), first, more):
        assert torch.equal(got, torch.cat([a, b], 2))


def test_cos_and_sin_of_other_strides(kernels):  # noqa: F811
    """Equal numbers in memory of another order are no reason to refuse."""
    c = cache(batch=1)
    k, v = tokens(1, 3, seed=1)
    wide = torch.ones(1, 3, 40)
    c.append(k, v, 0, tokens(1, 3, 4)[0], wide[..., :16], torch.ones(1, 3, 16))
    assert c.get_seq_length() == 3


@pytest.mark.parametrize("n", [1, 200])
def test_a_launch_that_fails(kernels, n):  # noqa: F811
    """Out of memory, say, for the rotated queries: the step can be made again, or another one."""
    c, first = _begun()
    for _ in range(2):
        before = state(c)
        kernels.fail = torch.OutOfMemoryError("no memory")
        with pytest.raises(torch.OutOfMemoryError):
            c.append(*tokens(2, n, seed=1), 0)
        assert state(c) == before
    more = tokens(2, 3, seed=2)
    c.append(*more, 0)
    for got, a, b in zip(held(c), first, more):
        assert torch.equal(got, torch.cat([a, b], 2))


def test_a_table_that_fails(kernels, monkeypatch):  # noqa: F811
    """No memory for a wider table: the pages that were taken go back."""
    c, first = _begun()
    before = state(c)
    real = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *a, **k: (_ for _ in ()).throw(torch.OutOfMemoryError("no memory")))
    with pytest.raises(torch.OutOfMemoryError):
        c.append(*tokens(2, 30, seed=1), 0)
    monkeypatch.setattr(torch, "zeros", real)
    assert state(c) == before


def test_a_later_layer_that_fails(kernels):  # noqa: F811
    """The step stays begun: the layers before have its tokens, and the layer's call can be made again."""
    c, first = _begun(layers=2)
    more = tokens(2, 5, seed=2)
    c.append(*more, 0)
    before = state(c)
    kernels.fail = RuntimeError("no")
    with pytest.raises(RuntimeError):
        c.append(*more, 1)
    assert state(c) == before
    c.append(*more, 1)
    for layer in range(2):
        for got, a, b in zip(held(c, layer), first, more):
            assert torch.equal(got, torch.cat([a, b], 2))
