"""Which form decode_attention_kv4 takes, as its workspace size shows it: the form of one workgroup a
head needs none, and holds a head's scores of at most 1024 rows and 16 query heads on the chip."""
import pytest

from deltaattention_amd import _native

ROWS = 1024


@pytest.mark.parametrize("units", [1, 8, 255, 256, 260, 767, 768, 769, 4096, 65535])
@pytest.mark.parametrize("G", [1, 4, 8, 16, 17, 64])
def test_one_workgroup_holds_its_rows(units, G):
    size = _native.lib().da_kv4_attention_workspace_size
    for capacity in (1, 31, 768, 769, 1023, 1024, 1025, 2048, 4096, 4097, 16384, 16385, 1 << 20, 1 << 24):
        for accumulate in (0, 1):
            n = size(units, G, 1, capacity, accumulate)
            if capacity > ROWS or (accumulate and G > 16):
                # sums of 128 dims and two statistics a query head; a score a row and query head
                least = 4 * units * G * (130 + accumulate * capacity)
                assert n >= least, (capacity, accumulate, n)
            elif capacity <= 768:
                assert n == 0, (capacity, accumulate, n)


@pytest.mark.parametrize("B,Hq,Hkv", [(96, 32, 8), (95, 32, 8), (1, 64, 1), (768, 16, 1)])
def test_workspace_grows_with_the_rows(B, Hq, Hkv):
    """A cache of more rows never needs less than a shorter one once it is past one workgroup's."""
    size = _native.lib().da_kv4_attention_workspace_size
    for accumulate in (0, 1):
        at = [size(B, Hq, Hkv, c, accumulate) for c in (1025, 2049, 4097, 65537)]
        assert at == sorted(at) and at[0] > 0
