"""The sizes of the launches of the 8-bit entry points and of the norm (host code,
no GPU): a launch counts its lanes in 32 bits, whatever sizes it is for."""

import ctypes

import pytest

from internal import _function

LANES = 1 << 32  # the first count that no launch can have


@pytest.mark.parametrize("blocks", [1, 16, 17, 393216, 2**24, 2**28 - 16, 2**28 - 15, 2**28, 2**28 + 1, 2**40, 2**62])
def test_quantize8(blocks):
    grid = _function("_ZN3ien14quantize8_gridEl", ctypes.c_long, restype=ctypes.c_uint)(blocks)
    assert 1 <= grid and grid * 256 < LANES
    assert grid == min(-(-blocks // 16), 1 << 20)  # one turn, but for more than 2 GiB of blocks
