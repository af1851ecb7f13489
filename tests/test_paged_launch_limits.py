"""Calls of the paged cache's operators that are larger than one launch may be."""
import pytest
import torch

from deltaattention_amd import _native
from test_paged_refusals import A, BF16, _append, _batch, _kv, _refused


def test_append_of_too_many_tokens():
    """A wave a token: 2^26 of them are 2^32 threads."""
    for T in (1 << 26, 1 << 28, 1 << 40):
        _refused(_append(T=T), -1, "2^26 tokens")
