"""rope_axes and qkv_rope_axes against their formulas in 64 bits."""
from __future__ import annotations

import pytest

from _request_cases import U, assert_within, rope as plain_rope

pytestmark = pytest.mark.gpu

# An angle's fraction of a revolution in [-1/2, 1/2], doubled, is rounded to fp32: off by at most u of 1, pi u of an
# angle; its position and frequency in 64 bits by 2^-51 revolutions for each unit of position (2^20 here: 2^-29 = u / 32
# of a circle, 0.2 u of an angle); sine and cosine themselves by 2 steps of their values, 4 u.
ANGLE = (3.15 + 0.2 + 4.0) * U
SAME = 1e-30


def _bound(torch, D, want, size):
    """A turned pair is off by 2 ANGLE of its size (each value by ANGLE of both terms, at most sqrt 2 of the size) and
    3 u of rounding; the norm by a sum's depth over D and 8 u of steps."""
    depth = -(-D // 64) + 8
    return (2 * ANGLE + 3 * U) * size + (depth / 2 + 8) * U * want.abs() + SAME


def _positions(torch, cuda, g, B, L, axes, fractional, far, batched):
    shape = (B, L, axes) if batched else (L, axes)
    p = torch.randint(-50, 1000, shape, generator=g, device=cuda)
    p[..., 0] += far
    return p.float() * 0.3125 if fractional else p.to(torch.int32)


CASES = [  # B, L, H, D, sections, theta, shared, interleaved, fractional, far, batched
    (1, 1, 1, 2, [1], 1e4, False, True, False, 0, False),
    (2, 1, 16, 64, [10, 11, 11], 1e4, False, True, False, 1000000, True),
    (1, 7, 3, 64, [32], 1e4, False, True, False, 0, False),
    (2, 9, 3, 64, [8, 12, 12], 1e4, True, False, False, 0, True),
    (2, 33, 5, 72, [18, 18], 100.0, False, False, True, 0, True),
    (3, 5, 2, 6, [1, 1, 1], 1e4, False, False, False, -1000000, True),
    (1, 130, 4, 128, [16, 24, 24], 1e4, False, True, True, 0, False),
    (2, 17, 7, 10, [0, 5], 10.0, False, True, False, 0, False),
    (1, 65, 2, 256, [64, 64], 1e6, True, False, False, 5000, True),
    (1, 3, 2, 512, [256], 1e4, False, True, False, 0, False),
    (1, 6, 3, 510, [100, 155], 1e4, False, False, True, 0, False),
    (2, 40, 1, 34, [5, 6, 6], 1e4, False, False, False, 0, True),
    (1, 1025, 24, 48, [8, 8, 8], 1e4, False, True, False, 0, False),
    (1, 20, 40, 96, [16, 16, 16], 1e4, False, True, False, 0, False),
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("normed", [False, True])
def test_one_tensor(cuda, hiplib, case, normed):
    import torch
    from tsplat.qkv import RopeAxes, rope_axes

    B, L, H, D, sections, theta, shared, inter, fractional, far, batched = case
    print(f"rope {case} {normed}", flush=True)
    g = torch.Generator(device=cuda).manual_seed(D)
    x = torch.randn(B, L, H, D, generator=g, device=cuda)
    gamma = torch.randn(H, D, generator=g, device=cuda) if normed else None
    pos = _positions(torch, cuda, g, B, L, len(sections), fractional, far, batched)
    rope = RopeAxes(D, sections, theta, shared=shared, interleaved=inter, device=cuda)
    want, size = plain_rope(torch, x, pos, sections, theta, shared, inter, gamma, 1e-12)
    got = rope_axes(x, pos, rope, gamma=gamma)
    assert_within(torch, got, want, _bound(torch, D, want, size), "bhld")
    other = rope_axes(x, pos, rope, gamma=gamma, out_bhld=False)
    assert torch.equal(other, got.transpose(1, 2))
    out = torch.full_like(got, float("nan"))
    assert rope_axes(x, pos, rope, gamma=gamma, out=out) is out and torch.equal(out, got)


@pytest.mark.parametrize("case", CASES, ids=str)
def test_qkv(cuda, hiplib, case):
    import torch
    from tsplat.qkv import RopeAxes, qkv_rope_axes, rope_axes

    B, L, H, D, sections, theta, shared, inter, fractional, far, batched = case
    print(f"qkv rope {case}", flush=True)
    g = torch.Generator(device=cuda).manual_seed(D + 1)
    qkv = torch.randn(B * L, 3 * H * D, generator=g, device=cuda)
    gammas = [torch.randn(H, D, generator=g, device=cuda) for _ in range(2)]
    pos = _positions(torch, cuda, g, B, L, len(sections), fractional, far, batched)
    rope = RopeAxes(D, sections, theta, shared=shared, interleaved=inter, device=cuda)
    q, k, v = qkv_rope_axes(qkv, pos, rope, *gammas, B, L, H)
    parts = qkv.view(B, L, 3, H, D)
    for got, i in ((q, 0), (k, 1)):
        want, size = plain_rope(torch, parts[:, :, i], pos, sections, theta, shared, inter, gammas[i], 1e-12)
        assert_within(torch, got, want, _bound(torch, D, want, size), f"part {i}")
        assert torch.equal(got, rope_axes(parts[:, :, i], pos, rope, gamma=gammas[i]))  # a strided view
    assert torch.equal(v, parts[:, :, 2].transpose(1, 2))
    q2, k2, _ = qkv_rope_axes(qkv, pos, rope, None, gammas[1], B, L, H)
    assert torch.equal(k2, k) and torch.equal(q2, rope_axes(parts[:, :, 0], pos, rope))


@pytest.mark.parametrize("D", [64, 72, 10])
@pytest.mark.parametrize("inter", [True, False])
def test_position_zero_and_zero_vectors(cuda, hiplib, D, inter):
    """No turn at position zero, bit for bit; a vector of zeros stays zeros under the norm; quarter turns are exact."""
    import torch
    from tsplat.qkv import RopeAxes, rope_axes

    x = torch.randn(2, 5, 3, D, device=cuda)
    rope = RopeAxes(D, [D // 2], interleaved=inter, device=cuda)
    pos = torch.zeros(5, 1, dtype=torch.int32, device=cuda)
    assert torch.equal(rope_axes(x, pos, rope, out_bhld=False), x)
    x[1, 3] = 0.0
    got = rope_axes(x, pos + 7, rope, gamma=torch.ones(3, D, device=cuda), out_bhld=False)
    assert torch.equal(got[1, 3], x[1, 3]) and torch.isfinite(got).all()
    rope.turns.fill_(0.25)  # a quarter of a revolution for each unit
    turned = rope_axes(x, pos + 4 * 1000003 + 1, rope, out_bhld=False)
    a, b = (x[..., 0::2], x[..., 1::2]) if inter else (x[..., :D // 2], x[..., D // 2:])
    ta, tb = (turned[..., 0::2], turned[..., 1::2]) if inter else (turned[..., :D // 2], turned[..., D // 2:])
    assert torch.equal(ta, -b) and torch.equal(tb, a)


def test_matches_the_frequency_table(cuda, hiplib):
    """One axis of token indices is what the packed QKV path reads from a table of cosines: the same result but for
    the table's own rounding."""
    import torch
    from tsplat.flow import rope_frequencies
    from tsplat.qkv import RopeAxes, qkv_rope_axes, qkv_rope_rmsnorm_pack

    B, L, H = 2, 50, 3
    g = torch.Generator(device=cuda).manual_seed(2)
    qkv = torch.randn(B * L, 3 * H * 64, generator=g, device=cuda)
    gammas = [1 + 0.1 * torch.randn(H, 64, generator=g, device=cuda) for _ in range(2)]
    freqs = rope_frequencies(torch, L, H, 1e4, cuda)
    want_q, want_k, want_v = qkv_rope_rmsnorm_pack(qkv, freqs, *gammas, B, L, H)
    pos = torch.arange(L, dtype=torch.int32, device=cuda)[:, None]
    q, k, v = qkv_rope_axes(qkv, pos, RopeAxes(64, [32], device=cuda), *gammas, B, L, H)
    size = torch.hypot(want_q[..., 0::2], want_q[..., 1::2]).repeat_interleave(2, -1)
    assert float(((q - want_q).abs() / size).max()) <= 4 * ANGLE + 30 * U
    want_k = want_k[..., :L].transpose(2, 3)
    size = torch.hypot(want_k[..., 0::2], want_k[..., 1::2]).repeat_interleave(2, -1)
    assert float(((k - want_k).abs() / size).max()) <= 8 * ANGLE + 60 * U
    assert torch.equal(v, want_v[..., :L].transpose(2, 3))


@pytest.mark.parametrize("D,H", [(64, 4), (72, 3), (10, 2)])
def test_strides(cuda, hiplib, D, H):
    """Heads, tokens and batch entries at strides of their own, unaligned starts; nothing beside them is read."""
    import torch
    from tsplat.qkv import RopeAxes, qkv_rope_axes, rope_axes

    B, L = 2, 11
    g = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randn(B, L, H, D, generator=g, device=cuda)
    gamma = torch.randn(H, D, generator=g, device=cuda)
    rope = RopeAxes(D, [D // 4, D // 2 - D // 4], interleaved=False, device=cuda)
    pos = torch.randint(0, 99, (L, 2), generator=g, device=cuda, dtype=torch.int32)
    want = rope_axes(x, pos, rope, gamma=gamma)
    for at, pad in ((0, 4), (1, 1), (2, 3), (4, 8)):
        wide = torch.full((B, L + 2, H + 1, D + pad + at), float("nan"), device=cuda)
        view = wide[:, 1:L + 1, :H, at:at + D]
        view.copy_(x)
        assert torch.equal(rope_axes(view, pos, rope, gamma=gamma), want)
    heads_first = torch.empty(B, H, L, D, device=cuda)
    heads_first.copy_(x.transpose(1, 2))
    assert torch.equal(rope_axes(heads_first.transpose(1, 2), pos, rope, gamma=gamma), want)
    guard = torch.full((B * H * L * D + 64,), 9.0, device=cuda)
    rope_axes(x, pos, rope, gamma=gamma, out=guard[32:-32].view(B, H, L, D))
    assert (guard[:32] == 9.0).all() and (guard[-32:] == 9.0).all()
    assert torch.equal(guard[32:-32].view(B, H, L, D), want)
    qkv = torch.randn(B * L, 3 * H * D, generator=g, device=cuda)
    wide = torch.full((B * L, 3 * H * D + 5), float("nan"), device=cuda)
    wide[:, 2:-3] = qkv
    for p, q in zip(qkv_rope_axes(wide[:, 2:-3], pos, rope, gamma, gamma, B, L, H),
                    qkv_rope_axes(qkv, pos, rope, gamma, gamma, B, L, H)):
        assert torch.equal(p, q)


def test_non_finite_vectors_stay_alone(cuda, hiplib):
    import torch
    from tsplat.qkv import RopeAxes, rope_axes

    x = torch.randn(1, 30, 5, 64, device=cuda)
    pos = torch.arange(60, dtype=torch.int32, device=cuda).view(30, 2)
    rope = RopeAxes(64, [16, 16], device=cuda)
    gamma = torch.ones(5, 64, device=cuda)
    clean = rope_axes(x, pos, rope, gamma=gamma)
    x[0, 4, 1, 7], x[0, 29, 4, 63] = float("nan"), float("inf")
    got = rope_axes(x, pos, rope, gamma=gamma)
    keep = torch.ones(5, 30, dtype=torch.bool, device=cuda)
    keep[1, 4] = keep[4, 29] = False
    assert torch.equal(got[0, keep], clean[0, keep])
    assert got[0, ~keep].isnan().any(-1).all()


def test_a_nan_is_its_vectors(cuda, hiplib):
    """A NaN makes its vector's norm one, and so the whole normed vector, as max(||y||, eps) of the formula does."""
    import torch
    from tsplat.qkv import RopeAxes, rope_axes

    for D in (6, 64, 72, 512):
        x = torch.randn(1, 9, 2, D, device=cuda)
        x[0, 3, 1, 5] = float("nan")
        pos = torch.arange(9, dtype=torch.int32, device=cuda)[:, None]
        got = rope_axes(x, pos, RopeAxes(D, [D // 2], device=cuda), gamma=torch.ones(2, D, device=cuda))
        assert got[0, 1, 3].isnan().all()
        assert int(got.isnan().sum()) == D


def test_more_tokens_than_a_grid_dimension(cuda, hiplib):
    """Workgroups past 65535 along the tokens: the last tokens come out as in a call of their own."""
    import torch
    from tsplat.qkv import RopeAxes, rope_axes

    L, D = 65536 * 4 + 9, 512  # four tokens a workgroup
    x = torch.randn(1, L, 1, D, device=cuda)
    pos = torch.arange(L, dtype=torch.int32, device=cuda)[:, None]
    rope = RopeAxes(D, [D // 2], device=cuda)
    got = rope_axes(x, pos, rope)
    for a, b in ((0, 64), (65535 * 4 - 20, 65535 * 4 + 20), (L - 30, L)):
        assert torch.equal(got[:, :, a:b], rope_axes(x[:, a:b], pos[a:b].contiguous(), rope))


def test_graph_and_stream(cuda, hiplib):
    import torch
    from tsplat.qkv import RopeAxes, qkv_rope_axes

    B, L, H = 1, 700, 4
    qkv = torch.randn(B * L, 3 * H * 64, device=cuda)
    pos = torch.arange(L, dtype=torch.float32, device=cuda)[:, None]
    rope = RopeAxes(64, [32], device=cuda)
    gamma = torch.ones(H, 64, device=cuda)
    want = qkv_rope_axes(qkv, pos, rope, gamma, gamma, B, L, H)
    outs = [torch.empty_like(t) for t in want]
    torch.cuda.synchronize(cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qkv_rope_axes(qkv, pos, rope, gamma, gamma, B, L, H, outs=outs)
    for _ in range(4):
        for o in outs:
            o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize(cuda)
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
        qkv_rope_axes(qkv, pos, rope, gamma, gamma, B, L, H)
    side = torch.cuda.Stream(device=cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        got = qkv_rope_axes(qkv, pos, rope, gamma, gamma, B, L, H)
    side.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(got, want))


def test_refusals(cuda, hiplib):
    import torch
    from tsplat.qkv import RopeAxes, qkv_rope_axes, rope_axes

    x = torch.randn(2, 5, 3, 64, device=cuda)
    pos = torch.zeros(5, 2, dtype=torch.int32, device=cuda)
    rope = RopeAxes(64, [16, 16], device=cuda)
    gamma = torch.ones(3, 64, device=cuda)
    for a, p, r, kw in ((x, pos.long(), rope, {}), (x, pos[:4], rope, {}), (x, pos[:, :1], rope, {}),
                        (x, pos.cpu(), rope, {}), (x, pos[None].expand(3, 5, 2).contiguous(), rope, {}),
                        (x, pos, RopeAxes(32, [8, 8], device=cuda), {}), (x, pos, None, {}),
                        (x, pos, RopeAxes(64, [16, 16], device="cpu"), {}), (x.half(), pos, rope, {}),
                        (x[0], pos, rope, {}), (x.transpose(2, 3), pos, rope, {}), (x[:1].expand(2, 5, 3, 64), pos, rope, {}),
                        (x, pos, rope, dict(gamma=gamma[:2])), (x, pos, rope, dict(gamma=gamma.double())),
                        (x, pos, rope, dict(eps=-1.0)), (x, pos, rope, dict(out=torch.empty(2, 5, 3, 64, device=cuda)))):
        with pytest.raises(ValueError):
            rope_axes(a, p, r, **kw)
    with pytest.raises(ValueError, match="backward"):
        rope_axes(x.clone().requires_grad_(), pos, rope)
    with pytest.raises(RuntimeError, match="-3"):
        rope_axes(x, pos, rope, out=x.view(2, 3, 5, 64))
    qkv = torch.randn(10, 3 * 3 * 64, device=cuda)
    with pytest.raises(ValueError):
        qkv_rope_axes(qkv, pos, rope, gamma, gamma, 2, 4, 3)
    with pytest.raises(ValueError):
        qkv_rope_axes(qkv[:, :-1], pos, rope, gamma, gamma, 2, 5, 3)
    with pytest.raises(ValueError):
        qkv_rope_axes(qkv, pos, rope, gamma, gamma, 2, 5, 3, outs=[x])
    one = torch.empty(2, 3, 5, 64, device=cuda)
    with pytest.raises(RuntimeError, match="-3"):
        qkv_rope_axes(qkv, pos, rope, gamma, gamma, 2, 5, 3, outs=[one, one, torch.empty_like(one)])
    none = rope_axes(torch.empty(2, 0, 3, 64, device=cuda), torch.zeros(0, 2, dtype=torch.int32, device=cuda), rope)
    assert none.shape == (2, 3, 0, 64)
