"""Stretched rotary frequencies at trained lengths where the slowest pair still turns."""

from __future__ import annotations

import math

import pytest
import torch

from spalmer_b200 import rotary_frequencies


@pytest.mark.parametrize("rotary_dim,base,length,factor", [(128, 10000.0, 131072, 4.0), (128, 10000.0, 65536, 16.0),
                                                           (64, 10000.0, 1 << 20, 8.0), (64, 500000.0, 8192, 8.0),
                                                           (128, 10000.0, 4096, 16.0)])
def test_yarn_blends_between_the_two_turn_counts(rotary_dim, base, length, factor):
    """Kept above 32 turns over the trained length, divided below one, linear in the pair's index in between,
    whether or not a pair turns as seldom as once."""

    freq, _ = rotary_frequencies(rotary_dim, base, scaling="yarn", factor=factor, original_length=length)
    plain, _ = rotary_frequencies(rotary_dim, base)
    pair = [rotary_dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
    low, high = math.floor(pair[0]), math.ceil(pair[1])
    share = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - low) / (high - low)).clamp(0, 1)  # divided
    assert torch.allclose(freq, plain * (share / factor + 1 - share), rtol=1e-13, atol=0)
    turns = length * plain / (2 * math.pi)
    assert torch.equal(freq[turns > 33], plain[turns > 33])
    assert torch.all(freq[turns > 1.0] > plain[turns > 1.0] / factor)  # none that turns more than once is divided whole
