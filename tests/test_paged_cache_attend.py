"""What PagedCache.attend takes (on the CPU, kernels replaced)."""
import pytest
import torch

from paged_cache_on_cpu import cache, kernels, tokens  # noqa: F401 (kernels: a fixture)


@pytest.mark.parametrize("n", [1, 5])
def test_queries_of_the_step_only(kernels, n):  # noqa: F811
    """More or fewer tokens than the step brought would attend as if they were others, or to nothing."""
    c = cache()
    with pytest.raises(RuntimeError, match="follows"):
        c.attend(torch.zeros(2 * n, 4, 16), 0)
    q = c.append(*tokens(2, n), 0, tokens(2, n, 4)[0])
    assert c.attend(q, 0).shape == (2, n, 4, 16)
    for bad in (q[:n], torch.cat([q, q]), torch.cat([q, q[:2]]), q[:0], q[None], q[0]):
        with pytest.raises(ValueError, match="tokens of 2 sequences"):
            c.attend(bad, 0)
