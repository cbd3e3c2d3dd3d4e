"""residual_norm against its formula in 64 bits."""
from __future__ import annotations

import itertools

import pytest

from _request_cases import U, residual_norm

pytestmark = pytest.mark.gpu


def _inputs(torch, cuda, B, L, C, seed, spread=1.0, mean=0.0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    x, h = r(B, L, C) * spread + mean, r(B, L, C)
    mod = r(B, 3 * C) * 0.3
    vectors = [1 + 0.1 * r(C), 0.1 * r(C), 1 + 0.1 * r(C), 0.1 * r(C)]
    return x, h, mod, vectors


def _norm_bound(torch, v, off, kind, weight, bias, eps):
    """(norm of v in 64 bits, how far an fp32 norm may be) where each value of v is off by at most `off`.

    First order, with s the root that divides and n the result: an error e of the input moves n_i by at most
    (|e_i| + rms(e) (1 + |n_i|)) / s; a sum of C values in chains of at most `depth` roundings is off by depth u of its
    terms' absolute sum, which is half of that in the root and, for the mean of the differences, at most depth u s; the
    subtractions, the root, the division and the product are 8 u of n; weight and bias round once each."""
    if kind is None:
        return v, off
    depth = -(-v.shape[-1] // 64) + 16
    d = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    s = torch.sqrt(d.square().mean(-1, keepdim=True) + eps)
    n = d / s
    bound = (off + off.square().mean(-1, keepdim=True).sqrt() * (1 + n.abs())) / s
    bound = bound + U * ((depth / 2 + 8) * n.abs() + (depth if kind == "layer" else 0))
    if weight is not None:
        n, bound = n * weight.double(), bound * weight.double().abs()
        bound = bound + U * n.abs()
    if bias is not None:
        n = n + bias.double()
        bound = bound + U * n.abs()
    return n, bound


def _bounds(torch, x, h, gate, c, post, pw, pb, pe, pre, w, b, e, scale, shift):
    """How far (x', y) may be: the norms' bounds, and a rounding for each product and sum between them."""
    v, off = _norm_bound(torch, h.double(), torch.zeros_like(h).double(), post, pw, pb, pe)
    if gate is not None:
        v, off = v * gate.double()[:, None], off * gate.double()[:, None].abs()
        off = off + U * v.abs()
    xc = c * x.double()
    off = off + U * (xc.abs() + (xc + v).abs())
    y, bound = _norm_bound(torch, xc + v, off, pre, w, b, e)
    if scale is not None:
        m, t = 1 + scale.double()[:, None], shift.double()[:, None]
        bound = bound * m.abs() + U * (2 * (y * m).abs() + (y * m + t).abs())
    return 1.01 * off + 1e-38, 1.01 * bound + 1e-38


def _run(torch, x, h, mod, vectors, post, pre, affine, gated, modulated, c=0.75, eps=1e-6, **more):
    from tsplat.block_ops import residual_norm as call

    C = x.shape[-1]
    gate = mod[:, :C] if gated else None
    scale, shift = (mod[:, C:2 * C], mod[:, 2 * C:]) if modulated else (None, None)
    pw, pb, w, b = vectors if affine else [None] * 4
    if post is None:
        pw = pb = None
    got = call(x, h, gate=gate, residual_scale=c, post_norm=post, post_weight=pw, post_bias=pb, post_eps=eps, norm=pre,
               weight=w, bias=b, eps=eps, scale=scale, shift=shift, **more)
    args = (x, h, gate, c, post, pw, pb, eps, pre, w, b, eps, scale, shift)
    return got, args


def _check(torch, x, h, mod, vectors, *flags, what="", **more):
    got, args = _run(torch, x, h, mod, vectors, *flags, **more)
    want = residual_norm(torch, *args)
    bounds = _bounds(torch, *args)
    for name, g, w, b in zip(("x'", "y"), got, want, bounds):
        assert torch.isfinite(g).all()
        worst = float(((g.double() - w).abs() / b).max())
        print(f"{what} {name}: {worst:.3f} of the bound", flush=True)
        assert worst <= 1.0, (what, name, worst)
    return got


FORMS = [f for f in itertools.product([None, "layer", "rms"], ["layer", "rms"], [False, True], [False, True],
                                      [False, True])]


@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(str(v) for v in f))
def test_every_form(cuda, hiplib, form):
    import torch

    for B, L, C in ((2, 5, 96), (1, 3, 1023)):
        print(f"form {form} {B} {L} {C}", flush=True)
        _check(torch, *_inputs(torch, cuda, B, L, C, 1, 3.0, 0.5), *form, what=f"{B}x{L}x{C}")


@pytest.mark.parametrize("C", [2, 3, 4, 63, 64, 65, 252, 256, 260, 511, 1000, 1024, 1028, 2044, 2048, 2050, 2052, 4095,
                               4096, 4100, 8191, 8192, 8196, 8200, 12288, 16384, 20001, 40000])
@pytest.mark.parametrize("post,pre", [("rms", "layer"), (None, "layer"), ("layer", "rms")])
def test_widths(cuda, hiplib, C, post, pre):
    import torch

    print(f"width {C} {post} {pre}", flush=True)
    _check(torch, *_inputs(torch, cuda, 2, 3, C, C, 2.0, -0.3), post, pre, True, True, True, what=f"C={C}")


@pytest.mark.parametrize("B,L,C", [(1, 1, 1024), (2, 1, 1024), (3, 4101, 64), (2, 1001, 260), (1, 12294, 1024),
                                   (70000, 1, 32)])
def test_rows(cuda, hiplib, B, L, C):
    import torch

    print(f"rows {B} {L} {C}", flush=True)
    _check(torch, *_inputs(torch, cuda, B, L, C, 7), "rms", "layer", True, True, True, what=f"{B}x{L}x{C}")


def test_one_column_and_constant_rows(cuda, hiplib):
    """No spread: a LayerNorm is its bias there, an RMS norm the sign; all zeros give zeros."""
    import torch
    from tsplat.block_ops import residual_norm as call

    x = torch.tensor([[3.0], [0.0], [-2.0]], device=cuda)
    out, y = call(x, torch.zeros_like(x), norm="layer", eps=1e-6)
    assert torch.equal(out, x) and torch.equal(y, torch.zeros_like(x))
    out, y = call(x, torch.zeros_like(x), norm="rms", eps=0.0 + 1e-30)
    assert torch.allclose(y[[0, 2]], torch.tensor([[1.0], [-1.0]], device=cuda), rtol=4 * U, atol=0)
    assert float(y[1]) == 0.0
    for C in (64, 1024, 1023, 9000, 20000):
        x = torch.full((3, C), 1234.5, device=cuda)
        _, y = call(x, torch.zeros_like(x), norm="layer", eps=1e-6)
        assert float(y.abs().max()) == 0.0
        _, y = call(torch.zeros_like(x), torch.zeros_like(x), norm="rms", post_norm="layer", eps=1e-6)
        assert float(y.abs().max()) == 0.0


@pytest.mark.parametrize("C", [64, 1023, 1024, 4096, 10000, 20000])
def test_rows_far_from_zero(cuda, hiplib, C):
    """A mean 2^14 times the deviation: the differences from it are exact in fp32 and the norm keeps them."""
    import torch

    g = torch.Generator(device=cuda).manual_seed(C)
    x = 16384.0 + torch.randint(-2048, 2048, (4, C), generator=g, device=cuda) / 2048.0
    from tsplat.block_ops import residual_norm as call

    out, y = call(x, torch.zeros_like(x), norm="layer", eps=1e-6)
    assert torch.equal(out, x)
    want = torch.nn.functional.layer_norm(x.double(), (C,), eps=1e-6)
    # values and deviation are near 1 (at most 1.8 times the deviation), the differences from the first mean exact, off
    # from the true mean's by a sum's depth of u of 16384: 1 at most, which the second mean takes away but for the depth
    # of u again; the root and the steps after it: (depth / 2 + 8) u of the value
    depth = C / 64 + 16
    assert float((y.double() - want).abs().max()) <= U * (2 * depth + (depth / 2 + 8) * 2)


@pytest.mark.parametrize("C", [96, 1023, 1024, 4096, 12000])
def test_in_place_strides_and_rows_behind(cuda, hiplib, C):
    import torch

    print(f"strides {C}", flush=True)
    B, L = 2, 7
    x, h, mod, vectors = _inputs(torch, cuda, B, L, C, 3)
    flags = ("rms", "layer", True, True, True)
    (want_x, want_y), _ = _run(torch, x, h, mod, vectors, *flags)
    a, b = x.clone(), h.clone()
    (got_x, got_y), _ = _run(torch, a, b, mod, vectors, *flags, out=a, normed=b)
    assert got_x is a and got_y is b and torch.equal(a, want_x) and torch.equal(b, want_y)
    for pad, at in ((1, 0), (4, 0), (5, 2), (8, 4)):
        wide = torch.full((4, B, L + 1, C + pad + at), 5.0, device=cuda)
        # (both batch entries at one stride of rows: the first L rows of each of B blocks do not qualify)
        flat = wide.view(4, B * (L + 1), -1)[:, :B * L, at:at + C]
        vx, vh, vo, vn = (flat[i].unflatten(0, (B, L)) for i in range(4))
        vx.copy_(x)
        vh.copy_(h)
        (got_x, got_y), _ = _run(torch, vx, vh, mod, vectors, *flags, out=vo, normed=vn)
        assert torch.equal(got_x, want_x) and torch.equal(got_y, want_y)
        for v in (vx, vh, vo, vn):
            v.fill_(5.0)
        assert (wide == 5.0).all()


def test_one_row_of_modulation_for_all(cuda, hiplib):
    import torch
    from tsplat.block_ops import residual_norm as call

    x, h, mod, _ = _inputs(torch, cuda, 3, 40, 130, 8)
    gate, scale, shift = (t.contiguous() for t in mod.chunk(3, 1))
    one = lambda t: t[:1]  # noqa: E731
    wide = lambda t: t[:1].expand(3, -1).contiguous()  # noqa: E731
    for g, s, t in ((one, one, one), (one, wide, wide), (wide, one, one), (one, None, None)):
        full = dict(gate=wide(gate)) | ({} if s is None else dict(scale=wide(scale), shift=wide(shift)))
        part = dict(gate=g(gate)) | ({} if s is None else dict(scale=s(scale), shift=t(shift)))
        for p, q in zip(call(x, h, **part), call(x, h, **full)):
            assert torch.equal(p, q)
    # per-batch rows of one, shared rows of the other
    want = call(x, h, gate=gate, scale=wide(scale), shift=wide(shift))
    got = call(x, h, gate=gate, scale=one(scale), shift=one(shift))
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_non_finite_rows_stay_alone(cuda, hiplib):
    import torch
    from tsplat.block_ops import residual_norm as call

    for C in (64, 1024, 1023, 9000):
        x, h, _, _ = _inputs(torch, cuda, 1, 37, C, 2)
        clean = call(x, h, post_norm="rms")
        x[0, 5, 3], h[0, 9, 1], x[0, 36, C - 1] = float("nan"), float("inf"), float("-inf")
        got = call(x, h, post_norm="rms")
        keep = torch.ones(37, dtype=torch.bool, device=cuda)
        keep[[5, 9, 36]] = False
        for p, q in zip(got, clean):
            assert torch.equal(p[0, keep], q[0, keep])
        assert got[1][0, ~keep].isnan().any(-1).all()


def test_graph_and_stream(cuda, hiplib):
    import torch

    x, h, mod, vectors = _inputs(torch, cuda, 2, 300, 256, 5)
    flags = ("layer", "rms", True, True, True)
    (want_x, want_y), _ = _run(torch, x, h, mod, vectors, *flags)
    out, normed = torch.empty_like(x), torch.empty_like(x)
    torch.cuda.synchronize(cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _run(torch, x, h, mod, vectors, *flags, out=out, normed=normed)
    for _ in range(4):
        out.fill_(float("nan"))
        normed.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize(cuda)
        assert torch.equal(out, want_x) and torch.equal(normed, want_y)
        _run(torch, x, h, mod, vectors, *flags)
    side = torch.cuda.Stream(device=cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        (got_x, got_y), _ = _run(torch, x, h, mod, vectors, *flags)
    side.synchronize()
    assert torch.equal(got_x, want_x) and torch.equal(got_y, want_y)


def test_refusals(cuda, hiplib):
    import torch
    from tsplat.block_ops import residual_norm as call

    x, h, mod, vectors = _inputs(torch, cuda, 2, 3, 8, 1)
    gate = mod[:, :8]
    for kw in (dict(gate=gate[:, :7]), dict(gate=mod[0, :8]), dict(scale=gate), dict(post_weight=vectors[0]),
               dict(weight=vectors[0][:7]), dict(weight=vectors[0].double()), dict(gate=gate.cpu()), dict(eps=-1.0),
               dict(norm="batch"), dict(post_norm="batch"), dict(scale=gate, shift=gate[:1]),
               dict(scale=gate, shift=gate.contiguous()), dict(out=x[:1]), dict(gate=gate.expand(2, 8)[[0, 1, 1]])):
        with pytest.raises(ValueError):
            call(x, h, **kw)
    for a, b in ((x, h[:, :2]), (x.half(), h.half()), (x, h.cpu()), (x.transpose(0, 1), h.transpose(0, 1).contiguous())):
        with pytest.raises(ValueError):
            call(a, b)
    with pytest.raises(ValueError, match="backward"):
        call(x.clone().requires_grad_(), h)
    for kw in (dict(out=h), dict(normed=x), dict(out=x, normed=x)):
        with pytest.raises(RuntimeError, match="-3"):
            call(x, h, **kw)
    empty = torch.empty(2, 0, 8, device=cuda)
    out, normed = call(empty, empty.clone(), gate=gate)
    assert out.shape == normed.shape == (2, 0, 8)


@pytest.mark.parametrize("C,share", [(8, 32), (130, 4)])
def test_more_rows_than_a_grid_dimension(cuda, hiplib, C, share):
    """Workgroups (of `share` rows) past 2^20 in a grid's first dimension: the last rows come out as in a call of
    their own."""
    import torch
    from tsplat.block_ops import residual_norm as call

    edge = share << 20
    M = edge + 11
    x, h = torch.randn(M, C, device=cuda), torch.randn(M, C, device=cuda)
    out, normed = call(x, h, post_norm="rms", eps=1e-5)
    for a, b in ((0, 9), (edge - 30, edge + 3), (M - 13, M)):
        want = call(x[a:b], h[a:b], post_norm="rms", eps=1e-5)
        assert torch.equal(out[a:b], want[0]) and torch.equal(normed[a:b], want[1])


@pytest.mark.parametrize("C", [1, 2, 5, 31, 32, 33, 48, 64, 66, 72, 100, 127, 128, 129])
@pytest.mark.parametrize("L", [1, 7, 33, 1001])
def test_narrow_rows(cuda, hiplib, C, L):
    """Several rows a wave, some of a workgroup's missing."""
    import torch

    x, h, mod, vectors = _inputs(torch, cuda, 3, L, C, C + L)
    for post, pre in (("rms", "layer"), ("layer", "rms"), (None, "layer")):
        _check(torch, x, h, mod, vectors, post, pre, True, True, True, what=f"{post} {pre}")


def test_a_row_of_the_most_columns(cuda, hiplib):
    """2^31 - 1 columns in place: a column index one step past the end does not fit 31 bits.  Values of +-1 whose sums
    are exact, so that the root's sum, the root, the division and the product are all that rounds: 3.5 u."""
    import torch
    from tsplat.block_ops import residual_norm as call

    C, half = 2 ** 31 - 1, 2 ** 30 - 1
    x, h = (torch.empty(C, device=cuda) for _ in range(2))
    for t in (x, h):
        t.fill_(0.5)
        t[:-1].view(half, 2)[:, 1] = -0.5
    print("2^31 - 1 columns", flush=True)
    out, normed = call(x[None], h[None], out=x[None], normed=h[None])
    torch.cuda.synchronize(cuda)
    want = 1 / (1 + 1e-6) ** 0.5
    for t, one, off in ((x, 1.0, 0.0), (h, want, 4 * U * want)):
        pairs = t[:-1].view(half, 2)
        for column, sign in ((pairs[:, 0], 1), (pairs[:, 1], -1), (t[-1:], 1)):
            low, high = (float(v) * sign for v in torch.aminmax(column))
            assert abs(low - one) <= off and abs(high - one) <= off, (sign, low, high)
