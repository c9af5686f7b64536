"""Rotary positions: head counts whose item counters would pass 31 bits."""

from __future__ import annotations

import ctypes

import pytest

UNSUPPORTED = -2


def test_heads_past_the_counters_are_refused():
    """The kernel adds up to 257 to a head index below the head count, in 32 bits
    (an index that wrapped around would address memory before the tensor)."""
    from ltx_amd import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("libltx_hip.so not built")
    lib = _lib.lib()
    few = _lib.RotaryRows(16, 0, 64, 64, 16, 0, 64, 64, 1)
    for heads in ((1 << 31) - 1, (1 << 31) - 200, (1 << 30) + 1):
        many = _lib.RotaryRows(16, 0, 64, 0, 16, 0, 64, 2, heads)
        for q, k in ((many, None), (few, many)):
            assert lib.ltx_rotary(ctypes.addressof(q), ctypes.addressof(k) if k else None, 0, 1, 1, 2, 2, 16, 0, 0, 16,
                                  1.0, 0, None) == UNSUPPORTED, heads
