"""A scale that fp32 holds and whose product with log2 e it does not hold is refused by the C entry, no GPU needed."""
from __future__ import annotations

import pytest

from test_cross_plan import _call, lib  # noqa: F401  (a fixture)


@pytest.mark.parametrize("scale,status", [(2.4e38, -2), (3.4e38, -2), (2.3e38, -6), (1e-45, -6)])
def test_scale(lib, scale, status):  # noqa: F811
    got = _call(lib, scale=scale)
    assert got == status or (status == -6 and got == -7)
