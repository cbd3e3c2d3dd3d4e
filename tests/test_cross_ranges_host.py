"""The bound that holds the cross attention's fp32 results feature by feature notices what a kernel could do wrong there:
mistakes planted in the 64-bit result, on the CPU."""
from __future__ import annotations

import pytest

from _cross_ranges import FEATURE, KINDS, feature_off, ranges, small_features


@pytest.mark.parametrize("kind", KINDS)
def test_mistakes_are_outside_the_bound(kind):
    import torch

    g = torch.Generator().manual_seed(12)
    q, k, v = (torch.randn(n, 2, 64, generator=g) for n in (60, 500, 500))
    v = small_features(kind, v)
    small = v.abs().amax(0) < 1e-3 * v.abs().amax()
    want, bound = ranges(torch, q, k, v, [60], [500])
    assert feature_off(torch, want.float(), want) <= FEATURE and bool(((want.float().double() - want).abs() <= bound).all())
    # all zero; v rounded to one step of a scale that all features share, which serves the large ones
    zeros = torch.where(small, 0.0, want)
    step = 2.0 ** -34 * float(v.abs().amax())
    shared = ranges(torch, q, k, (v.double() / step).round() * step, [60], [500])[0]
    for wrong in (zeros, shared):
        assert feature_off(torch, wrong, want) > FEATURE
    assert float(((zeros - want).abs() > bound)[:, small].double().mean()) > 0.9
    # 16-bit results
    assert feature_off(torch, want.bfloat16(), want) > FEATURE
