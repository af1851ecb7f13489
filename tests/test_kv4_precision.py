"""The statistical limits of kv4_precision on the CPU: the kernels' arithmetic passes them, and without any
one of its parts it does not."""
import pytest

import kv4_precision as P

SHAPES = [(1, 2, 4, 128, 600), (1, 1, 8, 64, 5000), (2, 2, 1, 96, 97)]
SIX = [(0, 2), (2, 0), (1, 1), (0, 1), (1, 0), (0, 0)]


def _rows(B, H, G, D, n, dtype):
    """Inputs whose k and v are values of the 4-bit format (here: bf16 is enough, the parts' products are exact)."""
    q, k, v, counts = P.attention_inputs(B, H, G, D, n, dtype, n + D)
    return q, k.bfloat16().float(), v.bfloat16().float(), counts


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_parts_are_seen(shape, dtype):
    ins = _rows(*shape, dtype)
    q_parts, p_parts = P.PARTS[dtype]
    P.assert_attention(*P.emulate(*ins, dtype, q_parts, p_parts), *ins, dtype)
    with pytest.raises(AssertionError, match="of the error without"):
        P.assert_attention(*P.emulate(*ins, dtype, q_parts, p_parts - 1), *ins, dtype)
    if q_parts > 1:
        out, mass = P.emulate(*ins, dtype, q_parts - 1, p_parts)
        with pytest.raises(AssertionError, match=r"q \(out\)"):
            P.assert_attention(out, None, *ins, dtype)
        good = P.emulate(*ins, dtype, q_parts, p_parts)[0]
        with pytest.raises(AssertionError, match=r"q \(mass\)"):
            P.assert_attention(good, mass, *ins, dtype)


@pytest.mark.parametrize("shape", [(1, 2, 1, 128, 1, 600), (1, 1, 4, 64, 7, 300), (2, 1, 2, 96, 40, 90)])
def test_mass_parts_are_seen(shape):
    q, k = P.mass_inputs(*shape, seed=shape[-1])
    P.assert_mass(P.emulate_mass(q, k, SIX), q, k)
    for lost in SIX:
        with pytest.raises(AssertionError):
            P.assert_mass(P.emulate_mass(q, k, [x for x in SIX if x != lost]), q, k)
