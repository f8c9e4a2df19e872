"""The rotations' table against fractions of a turn from exact arithmetic."""
from fractions import Fraction

import numpy as np
import pytest

import dragonwing_edge_rs_b200 as dw
from dragonwing_edge_rs_b200 import ops

pytestmark = pytest.mark.gpu
# 2 pi to 60 places
TWO_PI = Fraction(6283185307179586476925286766559005768394338798750211641949889, 10 ** 60)


@pytest.mark.parametrize("theta,pairs", [(1e4, 64), (5e5, 64), (1e6, 256), (100.0, 32), (-1e4, 64), (2.0 ** -40, 200)])
def test_turns_are_the_nearest(theta, pairs):
    """A turn's fraction is rounded once, by at most half a 2^-64, after a quotient that is off by two halves of a last
    place of 64 bits (the divisor's and its own), each at most 2^-64 of a fraction of up to 1 / 2 pi: 0.5 + 0.32."""
    sign = np.sign(theta)
    freqs = sign * np.abs(theta) ** (-np.arange(pairs) / pairs) if abs(theta) > 1 else np.linspace(theta, 1.0, pairs)
    with dw.CudaBackend(0) as be:
        table = be.download_array(ops.prepare_rope(be, freqs), np.uint64).reshape(3, pairs)
    for f, got, c, s in zip(freqs, *table[:1], *table[1:].view(np.float64)):
        want = Fraction(float(f)) / TWO_PI * 2 ** 64
        off = (int(got) - want) % 2 ** 64
        assert min(off, 2 ** 64 - off) <= Fraction(82, 100), (f, float(off))
        assert abs(c - np.cos(np.float64(f))) <= 2.0 ** -52 and abs(s - np.sin(np.float64(f))) <= 2.0 ** -52
