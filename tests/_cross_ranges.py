"""How far the cross attention of fp32 values may be from its definition where the values' sizes are unlike: the bound of
_cross_cases without what it grants every value by the largest of all.

A pair of fp16 values holds a value of v to 2^-23 of it and to 2^-25 of the scaled one.  The kernel keeps a feature only
where the largest of its scaled values among the states at hand is 2^-4 at least, which makes the latter 2^-21 of the
feature's largest value; else bf16 terms hold 2^-24 of each value.  Weights lose 2^-36 of the largest one."""
from __future__ import annotations

import math

from _cross_cases import LEAST, LOST, STEP, U


def ranges(torch, q, k, v, q_lengths, k_lengths, bias=None, scale=None):
    """(result, bound) [rows, heads, D] in 64 bits, fp32 accuracy for each feature by itself."""
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
            off = ((2 * D * (1 + 2.0 ** -5) + 6) * U + LOST["fp32"]) * scale * torch.bmm(
                qq.abs(), kk.abs().transpose(1, 2).contiguous()) + 2 * 2.0 ** -22
            if bias is not None:
                b = bias[keep].double()
                s = s + b
                off = off + 4 * U * (b.abs() + s.abs())
            top = s.amax(-1, keepdim=True)
            w = torch.exp(s - top)
            d = off + U * ((s - top).abs() + 18)
            total = w.sum(-1, keepdim=True)
            w = w / total
            wv = torch.bmm(w, vv.abs())
            w_off = w * torch.expm1(d)
            all_off = w_off.sum(-1, keepdim=True)
            moved = (torch.bmm(w_off, vv.abs()) + all_off * wv) / (1 - all_off.clamp(max=0.75))
            n = len(keep)
            moved = moved + (4 * (n + n // 32 + 16) * U + LOST["fp32"]) * wv
            moved = moved + 2.0 ** -21 * vv.abs().amax(1, keepdim=True) + 2.0 ** -36 * vv.abs().sum(1, keepdim=True) / total
            out[q0:q0 + nq] = torch.bmm(w, vv).transpose(0, 1)
            bound[q0:q0 + nq] = moved.transpose(0, 1)
        q0, k0 = q0 + nq, k0 + nk
    return out, 1.02 * bound + STEP["float32"] * (out.abs() + bound) + LEAST["float32"]


# A weight's error has either sign: scores of a few units, sums of D products of them, 2 U sqrt(D) = 9e-7 of a unit, the
# pairs' 2 * 2^-22, the exponent's and exponential's 24 U = 1.4e-6; in the root mean square below 3e-6, which a mean of
# values of either sign keeps relative to its own norm.  Values lose 2^-21 = 4.8e-7 of their feature's largest at most, four
# times their norm or so.
FEATURE = 1e-5


def feature_off(torch, got, want):
    """The largest relative error of a feature's results over rows and heads."""
    got, want = got.double().flatten(0, 1), want.flatten(0, 1)
    return float(((got - want).norm(dim=0) / want.norm(dim=0).clamp_min(1e-300)).max())


def small_features(kind, v):
    """v [states, heads, D] with features far below their neighbours."""
    if kind == "one":
        v[:, :, 9] *= 1e-9
    elif kind == "every fourth":
        v[:, :, ::4] *= 1e-7
    elif kind == "eight":
        v[:, :, 8:16] *= 1e-9
    elif kind == "lost":  # far below what a pair holds at all
        v[:, :, 5] *= 1e-20
    return v


KINDS = ["one", "every fourth", "eight", "lost"]
