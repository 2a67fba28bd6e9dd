"""The frequencies of rotary positions for longer contexts, pair by pair."""
import math

import pytest

from parameter_server_b200.ops import rotary


@pytest.mark.parametrize("dim,base,factor,trained,fast,slow", [(128, 10000.0, 4.0, 4096, 32.0, 1.0), (64, 500000.0, 8.0, 8192, 32.0, 1.0), (96, 10000.0, 2.5, 2048, 20.0, 2.0), (2, 10000.0, 4.0, 64, 32.0, 1.0)])
def test_yarn_goes_linearly_in_the_number_of_turns(dim, base, factor, trained, fast, slow):
    """Each value is off by the rounding of a handful of operations in 64 bits."""
    freqs, scale = rotary.rotary_frequencies(dim, base, scaling="yarn", factor=factor, trained_length=trained, fast=fast, slow=slow, device="cpu")
    between = 0
    for i, got in enumerate(freqs.tolist()):
        plain = math.exp(-2 * i / dim * math.log(base))
        turns = trained * plain / (2 * math.pi)
        share = min(max((turns - slow) / (fast - slow), 0.0), 1.0)   # of the plain frequency
        between += 0.0 < share < 1.0
        assert abs(got / (share * plain + (1 - share) * plain / factor) - 1) < 1e-13, i
    assert between > (0 if dim == 2 else dim // 16) and abs(scale - 1 - math.log(factor) / 10) < 1e-15
