"""cross_attention at the ends of its values' range, and where neighbouring features are of unlike sizes."""
from __future__ import annotations

import math

import pytest

from _cross_cases import cross
from _cross_ranges import FEATURE, KINDS, feature_off, ranges, small_features
from _request_cases import assert_within

pytestmark = pytest.mark.gpu

INF = math.inf


def _inputs(torch, cuda, rows, n, heads, D, dtype, seed, aligned=True):
    """q, k, v; unaligned: the same values in rows of an odd pitch, which take another kernel."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    made = [torch.randn(m, heads, D, generator=g, device=cuda).to(getattr(torch, dtype)) for m in (rows, n, n)]
    return made if aligned else [_unaligned(t) for t in made]


def _unaligned(t):
    wide = t.new_zeros(t.shape[0], t.shape[1], t.shape[2] + 1)
    wide[..., 1:] = t
    return wide[..., 1:]


def _plan(torch, cuda, rows, n, heads, D, dtype, precision="fp32"):
    from tsplat.cross_attention import CrossPlan

    return CrossPlan([rows], [n], heads, D, dtype=getattr(torch, dtype), precision=precision, device=cuda)


@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("q_size,k_size", [(1e-19, 1e-19), (1e-20, 1e-20), (1e-38, 1e-5), (1e-30, 1e-37), (1e-38, 1.0)])
def test_scores_next_to_zero(cuda, hiplib, q_size, k_size, D):
    """Scores that fp32 cannot tell from zero: the mean of the values, with a last block of states that is not full."""
    import torch
    from tsplat.cross_attention import cross_attention

    q, k, v = _inputs(torch, cuda, 300, 500, 2, D, "float32", 1)
    q, k = q * q_size, k * k_size
    q[7] = 0.0
    bias = torch.zeros(500, device=cuda)
    for b in (None, bias):
        want, bound = ranges(torch, q, k, v, [300], [500], b)
        got = cross_attention(q, k, v, _plan(torch, cuda, 300, 500, 2, D, "float32"), key_bias=b)
        assert_within(torch, got.double(), want, bound, "bias" if b is not None else "plain")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,size", [(2000, 1e32), (2000, 1e34), (2000, 1.5e35), (20000, 1e34)])
def test_sums_of_large_values(cuda, hiplib, n, size, D):
    """Equal scores over values whose sum fp32 holds: no weight above 1 may carry it past the type's range.  20000 states
    are cut into parts."""
    import torch
    from tsplat.cross_attention import cross_attention

    q, k, v = _inputs(torch, cuda, 300, n, 1, D, "float32", 2)
    q = torch.zeros_like(q)
    v = (1 + 0.1 * v) * size
    for b in (None, torch.zeros(n, device=cuda)):
        want, bound = ranges(torch, q, k, v, [300], [n], b)
        got = cross_attention(q, k, v, _plan(torch, cuda, 300, n, 1, D, "float32"), key_bias=b)
        assert_within(torch, got.double(), want, bound, "large")


@pytest.mark.parametrize("dtype,precision", [("float32", "fp32"), ("float32", "bf16x3"), ("float32", "bf16"),
                                             ("bfloat16", "fp32")])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("rows", [2, 100])
def test_sums_of_large_values_with_rising_scores(cuda, hiplib, rows, aligned, dtype, precision):
    """The same, with half of the states' scores 5.4 above the first ones', which a reference that lags behind the largest
    score makes weights of 2^7.8."""
    import torch
    from tsplat.cross_attention import cross_attention

    n = 2000
    q, k, v = _inputs(torch, cuda, rows, n, 1, 64, dtype, 3)
    q[:], k[:] = 0, 0
    q[..., 0] = 8.0
    k[:, :, 0] = torch.where(torch.arange(n, device=cuda) % 256 < 128, 0.0, 5.375)[:, None].to(k.dtype)
    v = ((1 + 0.1 * v.float()) * 1e35).to(v.dtype)
    if not aligned:
        q, k, v = (_unaligned(t) for t in (q, k, v))
    want, bound = cross(torch, q, k, v, [rows], [n], precision=precision)
    got = cross_attention(q, k, v, _plan(torch, cuda, rows, n, 1, 64, dtype, precision))
    assert bool(torch.isfinite(want).all())
    assert_within(torch, got.double(), want, bound, precision)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 96, 128])
def test_features_of_unlike_sizes(cuda, hiplib, kind, D):
    """A feature far below its neighbours keeps fp32's accuracy, whether or not its neighbours are small as well."""
    import torch
    from tsplat.cross_attention import cross_attention

    for rows, n, aligned in ((300, 500, True), (300, 500, False), (3, 500, True), (70, 4000, True)):
        q, k, v = _inputs(torch, cuda, rows, n, 2, D, "float32", 4)
        v = small_features(kind, v)
        if not aligned:
            q, k, v = (_unaligned(t) for t in (q, k, v))
        bias = torch.where(torch.arange(n, device=cuda) % 5 == 0, -INF, 0.0)
        plan = _plan(torch, cuda, rows, n, 2, D, "float32")
        for b in (None, bias):
            want, bound = ranges(torch, q, k, v, [rows], [n], b)
            got = cross_attention(q, k, v, plan, key_bias=b)
            assert_within(torch, got.double(), want, bound, kind)
            assert feature_off(torch, got, want) <= FEATURE


def test_values_of_unlike_sizes_by_feature(cuda, hiplib):
    """States of sizes from 1e-12 to 1e12, and a feature that is zero among the first states."""
    import torch
    from tsplat.cross_attention import cross_attention

    q, k, v = _inputs(torch, cuda, 300, 500, 2, 64, "float32", 5)
    plan = _plan(torch, cuda, 300, 500, 2, 64, "float32")
    steps = v * torch.logspace(-12, 12, 500, device=cuda)[:, None, None]
    late = v.clone()
    late[:200, :, 11], late[200:, :, 11] = 0.0, late[200:, :, 11] * 1e-9
    for values in (steps, late):
        want, bound = ranges(torch, q, k, values, [300], [500])
        got = cross_attention(q, k, values, plan)
        assert_within(torch, got.double(), want, bound, "by feature")
        assert feature_off(torch, got, want) <= FEATURE


@pytest.mark.parametrize("precision", ["fp32", "bf16x3"])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("rows", [2, 100])
def test_largest_finite_values(cuda, hiplib, rows, aligned, precision):
    """Values between bf16's largest and fp32's: finite ones, in q, k and v."""
    import torch
    from tsplat.cross_attention import cross_attention

    top = torch.finfo(torch.float32).max
    for n in (1, 70):
        q, k, v = _inputs(torch, cuda, rows, n, 2, 64, "float32", 6)
        v[:, :, 2], v[:, :, 5] = top / n, -3.4e38 / n
        v[0, :, 7] = top
        v[1:, :, 7] = 0.0
        k[:, :, 0], q[:, :, 0] = top, 0.0
        k[:, :, 1], q[:, :, 1] = 0.0, -top
        if not aligned:
            q, k, v = (_unaligned(t) for t in (q, k, v))
        # (scale * log2 e * top is 3.3997e38, above bf16's largest)
        scale = 0.6925
        want, bound = cross(torch, q, k, v, [rows], [n], scale=scale, precision=precision)
        got = cross_attention(q, k, v, _plan(torch, cuda, rows, n, 2, 64, "float32", precision), scale=scale).double()
        # A result that may be off by `bound` may round past fp32's largest where it lies closer to it than that: the value
        # top itself, whose weight and denominator are each rounded.  3.4e38 does not (2.8e35 away; 3.1 * 2^-16 of it: 1.6e34).
        past = torch.isinf(got) & (want.abs() + bound > top)
        assert bool((got[past].sign() == want[past].sign()).all()) and not past[..., 5].any()
        got = torch.where(past, want, got)
        assert bool(torch.isfinite(got).all())
        assert_within(torch, got, want, bound, precision)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows", [1, 100])
@pytest.mark.parametrize("aligned", [True, False])
def test_largest_bias(cuda, hiplib, aligned, rows, dtype):
    """A finite bias is never taken for an infinity: fp32's largest leaves its own state alone."""
    import torch
    from tsplat.cross_attention import cross_attention

    q, k, v = _inputs(torch, cuda, rows, 300, 2, 64, dtype, 7, aligned)
    plan = _plan(torch, cuda, rows, 300, 2, 64, dtype)
    for at, value in ((0, 2.4e38), (150, 3e38), (299, torch.finfo(torch.float32).max)):
        bias = torch.zeros(300, device=cuda)
        bias[at] = value
        got = cross_attention(q, k, v, plan, key_bias=bias).double()
        want = v[at].double().expand_as(got)
        # one weight, which division by itself makes 1 to 2 ulp, a pair's 2^-23 of the value, the result's rounding
        assert_within(torch, got, want, (torch.finfo(v.dtype).eps / 2 + 2.0 ** -21) * want.abs(), str(value))
        bias[at] = INF
        assert bool(torch.isnan(cross_attention(q, k, v, plan, key_bias=bias)).all())


def test_scale_whose_product_is_no_number(cuda, hiplib):
    """scale * log2 e has to be finite as well."""
    import torch
    from tsplat.cross_attention import cross_attention

    q, k, v = _inputs(torch, cuda, 40, 50, 2, 64, "float32", 8)
    plan = _plan(torch, cuda, 40, 50, 2, 64, "float32")
    q = torch.zeros_like(q)
    assert bool(torch.isfinite(cross_attention(q, k, v, plan, scale=2.3e38)).all())
    for scale in (2.4e38, 2.9e38):
        with pytest.raises(ValueError):
            cross_attention(q, k, v, plan, scale=scale)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows", [1, 100])
def test_smallest_scale(cuda, hiplib, rows, dtype):
    """Scores of zero, and states past the last one that still count for nothing: the values' mean."""
    import torch
    from tsplat.cross_attention import cross_attention

    q, k, v = _inputs(torch, cuda, rows, 50, 2, 64, dtype, 9)
    plan = _plan(torch, cuda, rows, 50, 2, 64, dtype)
    want, bound = cross(torch, q, k, v, [rows], [50], scale=1.4e-45)
    assert_within(torch, cross_attention(q, k, v, plan, scale=1.4e-45).double(), want, bound, dtype)


@pytest.mark.parametrize("D", [64, 128])
def test_small_query_features(cuda, hiplib, D):
    """Query features 2^-32 of the row's largest against keys 2^6 of the first states': two states count, and their
    difference is the small features' score."""
    import torch
    from tsplat.cross_attention import cross_attention

    # (so many states that a part holds 192 of them at least; scale * log2 e is 1 to 1e-7)
    n, late, rows, scale = 3200, 150, 64, 0.6931472
    q = torch.full((rows, 1, D), 100.49 * 2.0 ** -27, device=cuda)
    q[..., 0] = 4000.0
    k = torch.zeros(n, 1, D, device=cuda)
    k[:, :, 1:] = 1.0 / 64
    k[0, :, 1:] = 1.0
    k[1] = 0.0
    k[late, :, 1:] = 63.0
    v = torch.zeros(n, 1, D, device=cuda)
    v[1], v[late] = -1.0, 1.0
    bias = torch.full((n,), -200.0, device=cuda)
    bias[1] = bias[late] = 0.0
    s = scale * (q.double()[:, 0] * k.double()[late, 0]).sum(1)
    want = torch.tanh(s / 2)[:, None, None].expand(rows, 1, D)
    got = cross_attention(q, k, v, _plan(torch, cuda, rows, n, 1, D, "float32"), key_bias=bias, scale=scale).double()
    # In log2 units: 2^-22 each for q's and k's small values, half a step of 16 for each state's exponent, 2 D U of a score;
    # the exponential 1 ulp, and as much again for sums and the division.  The result moves by half of a score (in units of e).
    bound = 0.5 * (math.log(2) * (2 * 2.0 ** -22 + 2 * 2.0 ** -21) + 2 * D * 2.0 ** -24 * float(s.max()) + 8 * 2.0 ** -24)
    assert float((got - want).abs().max()) <= bound, (float((got - want).abs().max()), bound)


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("rows", [2, 100])
@pytest.mark.parametrize("size", [1e-33, 1e-36, 1e-40])
def test_smallest_values(cuda, hiplib, size, rows, aligned):
    """Values whose last bf16 term is subnormal, and subnormal ones: an absolute step of 2^-133 is what is left of them."""
    import torch
    from tsplat.cross_attention import cross_attention

    q, k, v = _inputs(torch, cuda, rows, 50, 2, 64, "float32", 10)
    v *= size
    if not aligned:
        q, k, v = (_unaligned(t) for t in (q, k, v))
    want, bound = ranges(torch, q, k, v, [rows], [50])
    got = cross_attention(q, k, v, _plan(torch, cuda, rows, 50, 2, 64, "float32"))
    # half of bf16's smallest step, 2^-134, of each value, whose weights add up to 1; half of fp32's, 2^-150, of each of 50
    # sums of them at weights of 2^-8: 50 * 2^-142 < 2^-136
    assert_within(torch, got.double(), want, bound + 2.0 ** -134 + 2.0 ** -136, str(size))


@pytest.mark.parametrize("at", [0, 150])
def test_values_far_below_the_first_ones(cuda, hiplib, at):
    """States that scaling by the first ones' largest would bring to zero are not zeros."""
    import torch
    from tsplat.cross_attention import cross_attention

    q, k, v = _inputs(torch, cuda, 100, 200, 2, 64, "float32", 11)
    v *= 1e-12
    v[at] = 1e38 if at == 0 else 1e31
    bias = torch.zeros(200, device=cuda)
    bias[at] = -300.0  # its weight is below 1e-120
    want, _ = ranges(torch, q, k, torch.where(bias[:, None, None] < 0, 0.0, v), [100], [200], bias)
    got = cross_attention(q, k, v, _plan(torch, cuda, 100, 200, 2, 64, "float32"), key_bias=bias)
    assert feature_off(torch, got, want) <= FEATURE
