"""The YaRN blend between its borders, from the definition by turns."""

from __future__ import annotations

import math

import numpy as np
import pytest


@pytest.mark.parametrize("d,theta,length,stretch,fast,slow", [(64, 10000.0, 4096, 16.0, 32.0, 1.0),
                                                              (128, 500000.0, 8192, 4.0, 32.0, 1.0),
                                                              (80, 10000.0, 2048, 8.0, 24.0, 2.0)])
def test_yarn_blend(d, theta, length, stretch, fast, slow):
    """Pairs with at least ``fast`` turns keep their frequency, from the last of them
    it falls linearly with the pair's number to 1 / stretch at the first pair with at
    most ``slow`` turns."""
    from ltx_amd.kernels.rope_ops import rotary_frequencies

    inv, factor = rotary_frequencies(d, theta, scaling="yarn", stretch=stretch, original_length=length,
                                     beta_fast=fast, beta_slow=slow, device="cpu")
    base = theta ** (-2 * np.arange(d // 2) / d)
    turns = length * base / (2 * math.pi)
    last, first = int(np.nonzero(turns >= fast)[0][-1]), int(np.nonzero(turns <= slow)[0][0])
    assert 0 < last < first - 3 and first < d // 2
    share = np.clip((np.arange(d // 2) - last) / (first - last), 0, 1)
    np.testing.assert_allclose(inv.numpy(), base * (1 - share + share / stretch), rtol=1e-12)
    assert factor == pytest.approx(0.1 * math.log(stretch) + 1, rel=1e-15)
