"""Frequencies of rotary positions where the ramp over a head's pairs does not lie among them.  On the CPU."""
import math

import numpy as np
import pytest


def place(part, base, length, turns):
    return part * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))


@pytest.mark.parametrize("part,base,length,low,high,factor", [
    (128, 10000.0, 131072, 1, 32, 4.0),     # the slowest pair makes 2.4 turns: the ramp would end at pair 70
    (64, 500.0, 65536, 1, 32, 8.0),
    (64, 10000.0, 10 ** 6, 0.5, 4, 2.0),
    (32, 100.0, 2 ** 31, 1, 2, 16.0),       # all pairs lie before it
    (64, 10000.0, 4096, 1, 32, 8.0),        # among the pairs
    (64, 10000.0, 5, 1, 32, 8.0),           # all but behind it
    (64, 10000.0, 3, 1, 2, 8.0),            # both ends before the first pair
])
def test_index_ramp(pkg, part, base, length, low, high, factor):
    f, _ = pkg.rotary_frequencies(part, base=base, scaling="index", factor=factor, original_length=length, low=low, high=high)
    plain = base ** (-2.0 * np.arange(part // 2) / part)
    first, last = max(0, math.floor(place(part, base, length, high))), math.ceil(place(part, base, length, low))
    ramp = np.clip((np.arange(part // 2) - first) / max(last - first, 0.001), 0, 1)
    assert np.allclose(f, plain * (1 - ramp) + plain / factor * ramp, rtol=1e-13)
    if last >= part // 2:  # more than `low` turns: not yet the full factor
        assert f[-1] > plain[-1] / factor * 1.01


@pytest.mark.parametrize("kw", [dict(part=2 ** 32 + 64), dict(part=-2 ** 32 + 64), dict(part=-2), dict(original_length=2 ** 32 + 64), dict(original_length=-2 ** 31)])
def test_numbers_beyond_32_bits_are_refused(pkg, kw):
    """A length of 2^32 + 64 is not one of 64."""
    with pytest.raises(pkg.InvalidArgumentError):
        pkg.rotary_frequencies(**{"part": 64, "scaling": "turns", "factor": 8.0, "original_length": 4096, **kw})
    pkg.rotary_frequencies(64, scaling="turns", factor=8.0, original_length=2 ** 32 - 1)


@pytest.mark.parametrize("factor,magnitude", [(0.5, 1.0), (1.0, 1.0), (1.5, 0.1 * math.log(1.5) + 1)])
def test_magnitude(pkg, factor, magnitude):
    got = pkg.rotary_frequencies(64, scaling="index", factor=factor, original_length=4096)[1]
    assert math.isclose(got, magnitude, rel_tol=2.0 ** -24) and (got == 1.0 or factor > 1)
