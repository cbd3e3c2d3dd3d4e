"""fp8_linear over every code and the ends of the scales: single products, which are exact."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu


def _all_codes(torch, cuda):
    """The 126 positive finite e4m3 values, and zero."""
    return torch.arange(127, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn).double()


def _pinned(torch, rows, power, cuda):
    """[rows, 256] of zeros but for 448 * 2^power in each block's first column."""
    x = torch.zeros(rows, 256, dtype=torch.float64, device=cuda)
    x[:, ::128] = 448.0 * 2.0 ** power
    return x


def _case(torch, cuda, M, N, x_power, w_power):
    """Rows of x with one code each besides the pins, all of them in turn with both signs; every row of w holds one code in
    all columns but the pins' (w's pins are the last column of each block, where x is zero)."""
    codes = _all_codes(torch, cuda)
    at = torch.arange(M, device=cuda)
    x = _pinned(torch, M, x_power, cuda)
    column = 1 + at % 120 + 128 * (at // 120 % 2)
    x[at, column] = codes[at * 5 % 127] * 2.0 ** x_power * torch.where(at % 2 == 0, 1.0, -1.0)
    n = torch.arange(N, device=cuda)
    w = (codes[n * 3 % 127] * 2.0 ** w_power * torch.where(n % 3 == 0, -1.0, 1.0))[:, None].repeat(1, 256)
    w[:, 127::128] = 448.0 * 2.0 ** w_power
    w[:, ::128] = 0.0
    picked = x.clone()
    picked[:, ::128] = 0.0
    return x.float(), w.float(), picked.sum(1)[:, None] * (codes[n * 3 % 127] * 2.0 ** w_power * torch.where(
        n % 3 == 0, -1.0, 1.0))


@pytest.mark.parametrize("M", [5, 40, 260])
@pytest.mark.parametrize("x_power,w_power", [(0, 0), (-20, 7), (119, -118), (-118, 119), (-60, -60), (-100, 110), (-117, 100),
                                             (-126, 118), (-127, 118), (118, -126), (118, -127), (-127, -10)])
def test_every_code_times_every_code(cuda, hiplib, M, x_power, w_power):
    import torch
    from tsplat.fp8 import fp8_linear, quantize_blocks

    x, w, want = _case(torch, cuda, M, 127, x_power, w_power)
    print(f"codes M={M} 2^{x_power} 2^{w_power}", flush=True)
    q, weight = quantize_blocks(x), quantize_blocks(w)
    assert bool((q.exponents == x_power + 127).all()) and bool((weight.exponents == w_power + 127).all())
    assert torch.equal(q.dequantize().double(), x.double()) and torch.equal(weight.dequantize().double(), w.double())
    got = fp8_linear(x, weight).double()
    # A code as bf16 is the value itself down to 2^-126, below that a multiple of 2^-133 (half a step: 2^-134), which the
    # smallest code, 2^-9, meets under a scale below 2^-117; a result is a multiple of 2^-149.
    least = 2.0 ** -134
    other_x, other_w = 448.0 * 2.0 ** x_power, 448.0 * 2.0 ** w_power
    bound = torch.zeros_like(want) + 2.0 ** -150
    if x_power < -117:
        bound += least * other_w
    if w_power < -117:
        bound += least * other_x
    wrong = (got - want).abs() > bound
    assert not wrong.any(), (int(wrong.sum()), float((got - want).abs().max()))
    if min(x_power, w_power) >= -117 and x_power + w_power >= -100:
        assert torch.equal(got, want)
    # 16-bit results of the same products, rounded once: bf16 has fp32's range
    got = fp8_linear(q, weight, out_dtype=torch.bfloat16).double()
    assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + bound + 2.0 ** -134).all())


def test_values_that_round_past_fp32(cuda, hiplib):
    """fp32 values from 248 * 2^120 on round to the code 256 under the scale 2^120: 2^128, which fp32 does not hold."""
    import torch
    from tsplat.fp8 import quantize_blocks

    x = torch.tensor([[247.0 * 2.0 ** 120, 249.0 * 2.0 ** 120, torch.finfo(torch.float32).max, 0.0]], device=cuda)
    q = quantize_blocks(x)
    assert q.codes.float().tolist() == [[240.0, 256.0, 256.0, 0.0]] and q.exponents.tolist() == [[247]]
    assert q.dequantize().tolist() == [[240.0 * 2.0 ** 120, math.inf, math.inf, 0.0]]
