"""Plain 64-bit forms of the 8-bit rows and the Linear on them, and how far the kernels may be from them.
U = 2^-24 is half a step of fp32 relative to the value."""
from __future__ import annotations

import math

U = 2.0 ** -24
BLOCK = 128
STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}  # half a step of the result's type
LEAST = {"float32": 2.0 ** -150, "bfloat16": 2.0 ** -134, "float16": 2.0 ** -25}  # half of its smallest value


def blocks(torch, x):
    """(code values [M, B, 128], exponents + 127 [M, B]) of the rows of x in 64 bits; NaN for what is not finite."""
    M, K = x.shape
    B = -(-K // BLOCK)
    v = torch.zeros(M, B * BLOCK, dtype=torch.float64, device=x.device)
    v[:, :K] = x.double()
    v = v.view(M, B, BLOCK)
    finite = torch.isfinite(v)
    top = torch.where(finite, v.abs(), 0.0).amax(-1)
    power = torch.tensor([2.0 ** i for i in range(-127, 128)], dtype=torch.float64, device=x.device)
    e = torch.searchsorted(448.0 * power, top).clamp(max=254)  # the first whose 448 reaches the largest
    e = torch.where(top == 0, 127, e)
    u = torch.where(finite, v, 0.0) / power[e][:, :, None]
    size = torch.frexp(u.abs().clamp_min(2.0 ** -6)).exponent - 1  # 2^size <= |u|
    fine = torch.tensor([2.0 ** (i - 3) for i in range(-6, 9)], dtype=torch.float64, device=x.device)
    step = fine[(size + 6).long()]
    code = (u / step).round() * step
    return torch.where(finite, code, math.nan), e


def values(torch, x):
    """What the 8-bit rows of x stand for, in 64 bits."""
    code, e = blocks(torch, x)
    power = torch.tensor([2.0 ** i for i in range(-127, 128)], dtype=torch.float64, device=x.device)
    return (code * power[e][:, :, None]).reshape(x.shape[0], -1)[:, :x.shape[1]]


def gelu(torch, y):
    return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))


def linear(torch, x, w, bias, activation, gate, residual, dtype):
    """(result, bound).  Codes' products are exact; a sum of K of them, each addition off by a step of fp32 at most
    (2 U; the matrix cores may cut instead of round), by 2 K U sum |terms|.  GELU's slope is below 1.13; its own
    arithmetic: u = y (1 + 0.044715 y^2) and the product with a constant 6 roundings of an argument |2 u| log2 e, of
    which y / (1 + e^-2u) keeps |2u| e^-|2u| < 0.4 for u > 0, times y for u < 0 no more, and 4 roundings of its own
    (exp2 and the reciprocal 1 ulp = 2 U each): 16 U (|y| + |y|^3 e^-|2u| ..) < 16 U |y| + 16 U.  Then one rounding
    each for the gate, the residual and the result's type.
    16-bit results of more than 64 rows: the 8-bit cores bring 8 neighbouring products to the largest one's exponent and
    cut them at 2^-13 of its power of two, so that 8 are off by 8 * 2^-13 of the largest, less than their sum."""
    xv, wv = values(torch, x), values(torch, w).t().contiguous()
    K = x.shape[1]
    y, bound = xv @ wv, 2 * (K + 4) * U * (xv.abs() @ wv.abs())
    if dtype != "float32" and x.shape[0] > 64:
        bound = bound + 2.0 ** -10 * (xv.abs() @ wv.abs())
    if bias is not None:
        y = y + bias.double()
        bound = bound + U * y.abs()
    if activation:
        bound = 1.13 * bound + 16 * U * (y.abs() + 1)
        y = gelu(torch, y)
    if gate is not None:
        g = gate.double().repeat_interleave(x.shape[0] // gate.shape[0], 0)
        y, bound = y * g, bound * g.abs() + U * (y * g).abs()
    if residual is not None:
        y = y + residual.double()
        bound = bound + U * y.abs()
    return y, 1.01 * bound + STEP[dtype] * (y.abs() + bound) + LEAST[dtype]


def norm_off(torch, got, want):
    return float((got.double() - want).norm() / want.norm().clamp_min(1e-300))


# The cuts above have either sign alike: 8 terms' are 2^-13 * max * sqrt(8 / 3) in the root mean square, and those of K / 8
# groups add in squares, as the K products do; the largest of 8 products is 3 times their root mean square or so, which
# makes 2^-13 * 1.63 * 3 / sqrt(8) < 2^-12 of the result's norm.
CUT = 2.0 ** -12
