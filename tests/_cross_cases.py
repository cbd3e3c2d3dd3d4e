"""The ragged cross attention in 64 bits, and how far the kernels may be from it.  U = 2^-24 is half a step of fp32."""
from __future__ import annotations

import math

U = 2.0 ** -24
STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}  # half a step of the type
LEAST = {"float32": 2.0 ** -150, "bfloat16": 2.0 ** -134, "float16": 2.0 ** -25}  # half of its smallest value
# What a product of fp32 factors loses relative to |a| |b|: bf16 terms hold 2^-8, 2^-16, 2^-24 of a factor, and the
# products of the terms i and j with i + j of the number of terms or more are left out.  Pairs of fp16 values hold a factor
# to 2^-23 (half a step of 2^-12 of what is left, which is 2^-11 at most) and leave out a product of 2^-11 by 2^-11: 2^-21.
LOST = {"fp32": 8.1 * 2.0 ** -24, "bf16x3": 3.1 * 2.0 ** -16, "bf16": 2.01 * 2.0 ** -8}


def cross(torch, q, k, v, q_lengths, k_lengths, bias=None, scale=None, precision="fp32"):
    """(result, bound) [rows, heads, D] in 64 bits.

    A score is a sum of D products, each addition off by 2 U of the sum of magnitudes at most (the matrix cores may cut
    instead of round); the smaller terms' products add 2^-8 of that.  Scale and log2 e join in 4 roundings, the bias in 3
    (its product with log2 e, the sum, the clamp to the type).  The exponent x - m is one rounding of at most
    |x - m| + 8, the exponential 1 ulp.  A relative error d of each weight moves the result by 2 d sum w |v|; the sums over
    n states (and one more for each of the parts that they are cut into, fewer than n / 32 + 8) by 2 U each addition, in the
    numerator and the denominator; a 16-bit weight is rounded by half a step, in the numerator only, and in fp16 by 2^-25
    of what is lifted by 2^7, 2^-32 of the largest weight.  fp32 values in pairs of fp16: 2^-22 more of a score (twice: k's
    small values and q's), 2^-25 of v scaled to 2^9 at least for its first tile's largest, 2^-25 of weights lifted by 2^11."""
    name = str(q.dtype).split(".")[-1]
    rows, heads, D = q.shape
    group = heads // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(rows, heads, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    q0 = k0 = 0
    for nq, nk in zip(q_lengths, k_lengths):
        keep = torch.arange(k0, k0 + nk, device=q.device)
        if bias is not None:
            keep = keep[bias[keep] != -math.inf]
        if nq and len(keep):
            qq = q[q0:q0 + nq].double().transpose(0, 1).contiguous()
            kk, vv = (t[keep].double().transpose(0, 1).repeat_interleave(group, 0).contiguous() for t in (k, v))
            s = scale * torch.bmm(qq, kk.transpose(1, 2).contiguous())
            size = scale * torch.bmm(qq.abs(), kk.abs().transpose(1, 2).contiguous())
            lost = LOST[precision] if name == "float32" else 0.0
            off = ((2 * D * (1 + 2.0 ** -5) + 6) * U + lost) * size
            if name == "float32" and precision == "fp32":
                off = off + 2 * 2.0 ** -22
            if bias is not None:
                b = bias[keep].double()
                s = s + b
                off = off + 4 * U * (b.abs() + s.abs())
            top = s.amax(-1, keepdim=True)
            w = torch.exp(s - top)
            # (log2 units: the exponent's size over ln 2)
            d = off + U * ((s - top).abs() + 18)
            total = w.sum(-1, keepdim=True)
            w = w / total
            o = torch.bmm(w, vv)
            wv = torch.bmm(w, vv.abs())
            n = len(keep)
            # each weight's own relative error, in the numerator and, averaged over the weights, in the denominator
            w_off = w * torch.expm1(d)
            all_off = w_off.sum(-1, keepdim=True)
            moved = (torch.bmm(w_off, vv.abs()) + all_off * wv) / (1 - all_off.clamp(max=0.75))
            moved = moved + 2 * (2 * (n + n // 32 + 16)) * U * wv
            if name != "float32":
                moved = moved + STEP[name] * wv
                if name == "float16":
                    moved = moved + 2.0 ** -32 * vv.abs().sum(1, keepdim=True) / total
            else:
                moved = moved + lost * wv
                if precision == "fp32":
                    moved = moved + 2.0 ** -34 * vv.abs().amax() + 2.0 ** -36 * vv.abs().sum(1, keepdim=True) / total
            out[q0:q0 + nq] = o.transpose(0, 1)
            bound[q0:q0 + nq] = moved.transpose(0, 1)
        q0, k0 = q0 + nq, k0 + nk
    return out, 1.02 * bound + STEP[name] * (out.abs() + bound) + LEAST[name]
