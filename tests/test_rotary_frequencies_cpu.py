"""ops.rotary_frequencies between the ends of its mixture, each frequency from the formula by itself: the share that is kept is linear in the turns that a pair makes in the original context."""
import math

import pytest
import torch

from randumb_amd import ops


@pytest.mark.parametrize("dim,base,factor,context,low,high", [(128, 10000.0, 8.0, 4096, 1.0, 32.0), (64, 500000.0, 4.0, 8192, 1.0, 32.0), (80, 10000.0, 2.5, 512, 2.0, 8.0),
                                                              (2, 10000.0, 4.0, 100, 1.0, 32.0), (32, 1.0, 4.0, 64, 1.0, 32.0)])
def test_parts(dim, base, factor, context, low, high):
    freq, scale = ops.rotary_frequencies(dim, base, scaling="parts", factor=factor, original_context=context, low=low, high=high)
    between = 0
    for i, got in enumerate(freq.tolist()):
        plain = base ** (-2 * i / dim)
        turns = context * plain / (2 * math.pi)
        kept = min(1.0, max(0.0, (turns - low) / (high - low)))
        between += 0.0 < kept < 1.0
        want = plain / factor + kept * (plain - plain / factor)
        assert abs(got - want) <= 2.0**-24 * want * (1 + 1e-6)   # rounded once, to fp32
    assert between or dim <= 2
    assert math.isclose(scale, 0.1 * math.log(factor) + 1.0)


def test_ends_of_the_mixture():
    """A pair of exactly ``low`` turns is divided, one of ``high`` turns kept."""
    context = 2 * math.pi * 32.0
    freq, _ = ops.rotary_frequencies(4, 1024.0, scaling="parts", factor=4.0, original_context=context, low=1.0, high=32.0)   # 32 turns, and one
    assert freq.tolist() == [1.0, 1.0 / 32 / 4]
