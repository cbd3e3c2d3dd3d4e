"""Plain 64-bit forms of the request operators, and how far fp32 may be from
them.  u = 2^-24 is half a step of fp32 relative to the value."""
from __future__ import annotations

import math

U = 2.0 ** -24


def low_rank(torch, y, x, rows, adapters):
    """(result, bound): adapters {slot: (down, up, scale)}.  A sum of n products in any order is off by at most
    n u sum |terms| (first order); 6 u more for the split of an operand and what its smallest products leave out."""
    out, bound = y.double().clone(), U * y.double().abs()
    K = x.shape[1]
    for a, (down, up, scale) in adapters.items():
        at = (rows == a).nonzero()[:, 0]
        if len(at) == 0:
            continue
        d, v, xs = down.double().t().contiguous(), up.double().t().contiguous(), x[at].double()
        R = d.shape[1]
        t, t_abs = xs @ d, xs.abs() @ d.abs()
        delta = scale * (t @ v)
        out[at] += delta
        reach = abs(scale) * (t_abs @ v.abs())
        bound[at] += U * ((K + R + 16) * reach + delta.abs() + out[at].abs())
    return out, 1.01 * bound


def norm(torch, v, kind, weight, bias, eps):
    if kind is None:
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    v = v if weight is None else v * weight.double()
    return v if bias is None else v + bias.double()


def residual_norm(torch, x, h, gate, c, post, pw, pb, pe, pre, w, b, e, scale, shift):
    """(x', y) in 64 bits; gate, scale, shift: [B, C] or None for x [B, L, C]."""
    v = norm(torch, h.double(), post, pw, pb, pe)
    v = v if gate is None else v * gate.double()[:, None]
    x = c * x.double() + v
    y = norm(torch, x, pre, w, b, e)
    return x, y if scale is None else y * (1 + scale.double()[:, None]) + shift.double()[:, None]


def rope(torch, x, positions, sections, theta, shared, interleaved, gamma, eps):
    """x [B, L, H, D] -> ([B, H, L, D] in 64 bits, the size of each pair after the norm, as an error scale)."""
    B, L, H, D = x.shape
    P = D // 2
    axis = torch.tensor([i for i, n in enumerate(sections) for _ in range(n)], device=x.device)
    ramp = [theta ** (-p / P) for p in range(P)] if shared else [theta ** (-j / n) for n in sections for j in range(n)]
    pos = positions.double().reshape(-1, L, len(sections))[..., axis]
    t = (pos * torch.tensor(ramp, dtype=torch.float64, device=x.device))[:, :, None]
    x = x.double()
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :P], x[..., P:])
    re, im = a * t.cos() - b * t.sin(), a * t.sin() + b * t.cos()
    size = torch.hypot(a, b)

    def join(p, q):
        return torch.stack((p, q), -1).flatten(-2) if interleaved else torch.cat((p, q), -1)

    out, size = join(re, im), join(size, size)
    if gamma is not None:
        k = math.sqrt(D) / x.norm(dim=-1, keepdim=True).clamp_min(eps) * gamma.double()
        out, size = out * k, size * k.abs()
    return out.transpose(1, 2), size.transpose(1, 2)


def assert_within(torch, got, want, bound, what=""):
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    assert torch.isfinite(want).all() and torch.isfinite(bound).all(), what
    off = (got.double() - want).abs()
    # (a zero that is kept as it is has a bound of zero and is off by none: 0 / 0 is no fault)
    worst = float(torch.where(off == 0, off, off / bound).max()) if off.numel() else 0.0
    print(f"{what}: {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0, (what, worst)
