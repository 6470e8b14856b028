"""The bound that the 8-bit attention is held to on a GPU (`test_gpu_accuracy8.py`) tells what it is there to tell: weights of
22 bits stay far inside it, weights that lost their low part, or have another's, are far outside.  Nothing here runs a kernel."""
import pytest
import torch

from tests import accuracy8 as A
from tests import cache8_ref as R

CASES = [(2, 4, 128, "e4m3"), (2, 3, 64, "int8"), (1, 8, 128, "int8"), (2, 5, 64, "e4m3"), (1, 16, 128, "e4m3"), (1, 12, 64, "int8")]


def _over(c, Hkv, G, weights):
    """Largest error of each sequence over its bound."""
    exact, mag = A.emulate(c, Hkv, G, lambda p: p)
    got, _ = A.emulate(c, Hkv, G, weights)
    return [float(((got[b] - exact[b]).abs() / (A.rel_bound(n) * mag[b])).max()) for b, n in enumerate(A.LENS)]


@pytest.mark.parametrize("Hkv,G,D,kind", CASES)
def test_the_bound_tells_22_bits_from_11(Hkv, G, D, kind):
    c = A.inputs(Hkv, G, D, kind, torch.bfloat16, seed=G * D)
    assert max(_over(c, Hkv, G, A.two_parts)) < 0.2
    for wrong in (A.one_part, A.low_part_of_half_the_tokens) + ((A.low_part_of_the_next_head,) if G > 1 else ()):
        over = _over(c, Hkv, G, wrong)
        # (one token: its weight is 1 in any number of bits)
        assert all(x > 2 for x, n in zip(over, A.LENS) if n > 1), (wrong.__name__, over)


@pytest.mark.parametrize("Hkv,G,D,kind", CASES)
def test_the_scores_are_exact_in_fp32(Hkv, G, D, kind):
    c = A.inputs(Hkv, G, D, kind, torch.float16, seed=G * D)
    for b, n in enumerate(A.LENS):
        x = A.log2_scores(c, b, 0, G)
        assert (x * 64 == (x * 64).round()).all() and x.abs().max() < 32 and (n == 1 or x.std() > 0.5)
    # and the emulation is the attention
    ref = R.decode_f64(c["q"], c["k"].float() if kind == "e4m3" else c["k"], c["v"].float() if kind == "e4m3" else c["v"],
                       c["ks"], c["vs"], A.SCALE, A.LENS)
    out, mag = A.emulate(c, Hkv, G, lambda p: p)
    assert ((out - ref["out"]).abs() <= 1e-12 * ref["mag"]).all() and torch.allclose(mag, ref["mag"], rtol=1e-12)
