"""The largest calls that a launch takes, on the CPU: one token more is refused by its size."""
import ctypes

import pytest

import breadv2_amd as B
from breadv2_amd import _lib

P = 0x1000  # an aligned address that is never read


@pytest.mark.parametrize("E", [300, 1024])
def test_route_select_refuses_what_no_launch_holds(E):
    r = _lib.RouteRuleDesc(None, 0, 1, 1, 1, 1, 1.0)
    for T in ((1 << 26) - 3, 1 << 26):
        assert -(-T // 4) * 256 >= 1 << 32
        assert B.lib.bread_route_select(ctypes.byref(r), P, 0, E, 8, T, P, P, None) == _lib.ERR_SHAPE
