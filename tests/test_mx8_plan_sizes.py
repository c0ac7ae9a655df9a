"""Plans are given for the sizes that the products take, and for no others."""

from __future__ import annotations

import ctypes

import pytest


@pytest.mark.parametrize("size", [((1 << 20) + 1, 32, 8, 0), (1 << 32 | 5, 32, 8, 0), (5, (1 << 20) + 32, 8, 0),
                                  (5, 32, (1 << 24) + 1, 0), (5, 32, 8, (1 << 24) + 1), (5, 32, 8, 1 << 32)])
def test_sizes_past_the_products_limits(size):
    from dsv41 import _abi
    with pytest.raises(ValueError, match="2\\^20"):
        _abi.linear_mx8_plan(*size)
    if max(size) < 1 << 31:
        plan = (ctypes.c_int32 * 4)()
        assert _abi.lib().dsv41_linear_mx8_plan(*size, plan) == -3 and b"2^24" in _abi.lib().dsv41_last_error_string()


def test_the_largest_sizes():
    from dsv41 import _abi
    for size in [(1 << 20, 32, 8, 0), (1, 1 << 20, 8, 0), (1, 32, 1 << 24, 1 << 24), (1 << 20, 1 << 20, 1 << 24, 1 << 24)]:
        assert _abi.linear_mx8_plan(*size).tile_rows > 0
