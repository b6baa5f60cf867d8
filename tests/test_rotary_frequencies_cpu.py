"""The frequencies of rotary positions, pair by pair, against their formulas written out."""
import math

import pytest

from pth_flash_attn_b200.kv8 import rotary_frequencies


@pytest.mark.parametrize("dims,base", [(64, 10000.0), (128, 1e6), (2, 10000.0), (96, 500.0)])
def test_plain_and_scaled(dims, base):
    plain, scale = rotary_frequencies(dims, base)
    linear, _ = rotary_frequencies(dims, base, scaling="linear", factor=4.0)
    ntk, _ = rotary_frequencies(dims, base, scaling="ntk", factor=4.0)
    assert scale == 1.0
    for i in range(dims // 2):
        assert float(plain[i]) == pytest.approx(base ** (-2 * i / dims), rel=1e-13)
        assert float(linear[i]) == pytest.approx(base ** (-2 * i / dims) / 4.0, rel=1e-13)
        if dims > 2:   # the fastest as before, the slowest four times slower, geometric between them
            assert float(ntk[i]) == pytest.approx(base ** (-2 * i / dims) * 4.0 ** (-2 * i / (dims - 2)), rel=1e-12)


@pytest.mark.parametrize("dims,base,factor,trained,fast,slow", [(64, 10000.0, 8.0, 4096, 32.0, 1.0), (128, 1e6, 16.0, 8192, 32.0, 1.0), (96, 10000.0, 2.0, 2048, 8.0, 2.0)])
def test_yarn_blends_linearly_in_the_index(dims, base, factor, trained, fast, slow):
    """From the floor of the index that turns `fast` times over the trained length to the ceiling of the one that turns `slow` times."""
    f, scale = rotary_frequencies(dims, base, scaling="yarn", factor=factor, trained=trained, fast=fast, slow=slow)
    assert scale == pytest.approx(0.1 * math.log(factor) + 1.0)

    def at(turns):   # i with trained base^(-2 i / dims) / (2 pi) = turns
        return dims / 2 * math.log(trained / (2 * math.pi * turns), base)

    low, high = max(0, math.floor(at(fast))), min(dims - 1, math.ceil(at(slow)))
    assert 0 <= low < high
    for i in range(dims // 2):
        plain, slower = base ** (-2 * i / dims), min(1.0, max(0.0, (i - low) / (high - low)))
        assert float(f[i]) == pytest.approx(plain * (1 - slower) + plain / factor * slower, rel=1e-12)
