"""Headers whose own numbers no plan has, no GPU needed: sizes that would pass 64 bits or a launch are refused, not
computed with."""
from __future__ import annotations

import ctypes

import pytest

from test_cross_plan import INTS, _call, lib, make  # noqa: F401  (lib is a fixture)

TOP = 2 ** 31 - 1


@pytest.mark.parametrize("change", [{7: TOP, 8: TOP}, {7: 65536, 8: 65536}, {7: 65535, 8: 65535}, {12: 2}, {12: -1},
                                    {7: 4, 8: 8}])
def test_refused(lib, change):  # noqa: F811
    n = 300  # one row and state each: 300 items, of which 65535 key heads would make more threads than a launch has
    header = make(lib, [1] * n, [300] * n, 4, 2)[:INTS]
    assert header[2] >= n and header[4] > 0
    for at, value in change.items():
        header[at] = value
    h = (ctypes.c_int32 * INTS)(*header)
    assert lib.tsplat_cross_scratch_bytes(h) == 0
    assert _call(lib, header=h) == -2
