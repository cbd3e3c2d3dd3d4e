"""cross_attention against its definition in 64 bits: lengths from none to thousands, heads of odd sizes and shared key
heads, biases that mask, strides and alignment, memory beside what is written, graphs and streams."""
from __future__ import annotations

import math

import pytest

from _cross_cases import cross
from _request_cases import assert_within

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16", "float16"]
INF = math.inf

#        queries, keys, heads, key heads, head size
CASES = [([1], [1], 1, 1, 1), ([1], [2], 1, 1, 64), ([3], [5], 2, 1, 7), ([1, 1], [33, 0], 2, 2, 8),
         ([1, 1, 1], [129, 1, 700], 8, 2, 128), ([5, 0, 3], [64, 9, 31], 4, 4, 64), ([33], [32], 1, 1, 32),
         ([31, 32, 33], [31, 33, 65], 2, 2, 72), ([129, 1], [127, 300], 6, 2, 40), ([257], [1], 3, 3, 96),
         ([130, 70, 0, 1], [0, 193, 5, 1025], 4, 1, 97), ([300], [260], 2, 2, 128), ([65, 2], [513, 70], 16, 2, 24),
         ([1], [3001], 1, 1, 64), ([8], [2049], 4, 1, 96), ([700, 40], [100, 2500], 1, 1, 64),
         ([0, 0], [4, 0], 2, 1, 16), ([], [], 2, 2, 64)]


def _inputs(torch, cuda, queries, keys, heads, kv_heads, D, dtype, seed, extra=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    dt = getattr(torch, dtype)
    q = torch.randn(sum(queries) + extra, heads, D, generator=g, device=cuda).to(dt)
    kv = torch.randn(sum(keys) + extra, 2, kv_heads, D, generator=g, device=cuda).to(dt)
    bias = torch.randn(sum(keys) + extra, generator=g, device=cuda)
    return q, kv[:, 0], kv[:, 1], bias, g


def _plan(torch, cuda, queries, keys, heads, kv_heads, D, dtype, precision="fp32"):
    from tsplat.cross_attention import CrossPlan

    return CrossPlan(queries, keys, heads, D, kv_heads=kv_heads, dtype=getattr(torch, dtype), precision=precision,
                     device=cuda)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CASES, ids=lambda c: "{}x{}_h{}-{}x{}".format(*c).replace(" ", ""))
def test_values(cuda, hiplib, case, dtype):
    import torch
    from tsplat.cross_attention import cross_attention

    queries, keys, heads, kv_heads, D = case
    print(f"cross {case} {dtype}", flush=True)
    q, k, v, bias, g = _inputs(torch, cuda, queries, keys, heads, kv_heads, D, dtype, D + len(queries))
    plan = _plan(torch, cuda, queries, keys, heads, kv_heads, D, dtype)
    bias[torch.rand(len(bias), generator=g, device=cuda) < 0.3] = -INF
    for b in (None, bias):
        want, bound = cross(torch, q, k, v, queries, keys, b)
        got = cross_attention(q, k, v, plan, key_bias=b)
        assert got.dtype is q.dtype
        assert_within(torch, got.double(), want, bound, "bias" if b is not None else "plain")
        assert torch.equal(got, cross_attention(q, k, v, plan, key_bias=b))
    want, bound = cross(torch, q, k, v, queries, keys, None, 0.3)
    assert_within(torch, cross_attention(q, k, v, plan, scale=0.3).double(), want, bound, "scale")


@pytest.mark.parametrize("precision", ["bf16x3", "bf16"])
@pytest.mark.parametrize("case", CASES[:16:3] + [CASES[7], CASES[10], CASES[14]],
                         ids=lambda c: "{}x{}_h{}-{}x{}".format(*c).replace(" ", ""))
def test_precisions(cuda, hiplib, case, precision):
    import torch
    from tsplat.cross_attention import cross_attention

    queries, keys, heads, kv_heads, D = case
    print(f"cross {case} {precision}", flush=True)
    q, k, v, bias, g = _inputs(torch, cuda, queries, keys, heads, kv_heads, D, "float32", 3)
    plan = _plan(torch, cuda, queries, keys, heads, kv_heads, D, "float32", precision)
    for b in (None, bias):
        want, bound = cross(torch, q, k, v, queries, keys, b, precision=precision)
        assert_within(torch, cross_attention(q, k, v, plan, key_bias=b).double(), want, bound, precision)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,heads,D", [(1, 1001, 16, 64), (40, 1001, 16, 64), (300, 200, 4, 96), (1, 3000, 32, 128),
                                            (150, 500, 6, 100)])
def test_every_state_counts_once(cuda, hiplib, rows, n, heads, D, dtype):
    """Equal scores, and values that are 1 for one state of each column: every result is 1 / n."""
    import torch
    from tsplat.cross_attention import cross_attention

    dt = getattr(torch, dtype)
    q = torch.zeros(rows, heads, D, device=cuda, dtype=dt)
    k = torch.randn(n, heads, D, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda).to(dt)
    at = torch.arange(heads * D, device=cuda) % n
    v = torch.zeros(n, heads * D, device=cuda, dtype=dt)
    v[at, torch.arange(heads * D, device=cuda)] = 1
    out = cross_attention(q, k, v.view(n, heads, D), _plan(torch, cuda, [rows], [n], heads, heads, D, dtype))
    # weights of 1 and their sums are exact; a division (1 ulp), a product and the result's rounding
    assert float((out.double() * n - 1).abs().max()) <= torch.finfo(dt).eps / 2 + 4 * 2.0 ** -24


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 200])
def test_many_small_weights(cuda, hiplib, rows, dtype):
    """One state of weight 1, thousands of 2^-20 and of 2^-26 each: their sum is not lost."""
    import torch
    from tsplat.cross_attention import cross_attention

    dt = getattr(torch, dtype)
    for power, n in ((20, 9000), (26, 30000)):
        q = torch.zeros(rows, 1, 64, device=cuda, dtype=dt)
        q[..., 0] = 8.0
        k = torch.zeros(n + 1, 1, 64, device=cuda, dtype=dt)
        k[1:, 0, 0] = -power * math.log(2)
        k[n // 2], k[0] = k[0].clone(), k[1].clone()
        v = torch.zeros(n + 1, 1, 64, device=cuda, dtype=dt)
        v[:, :, 1] = 1.0
        v[n // 2, 0, 1], v[n // 2, 0, 0] = 0.0, 1.0
        plan = _plan(torch, cuda, [rows], [n + 1], 1, 1, 64, dtype)
        want, bound = cross(torch, q, k, v, [rows], [n + 1])
        got = cross_attention(q, k, v, plan).double()
        assert_within(torch, got, want, bound, f"2^-{power}")
        assert float((got - want)[..., 1].abs().max()) <= 0.01 * float(want[..., 1].max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [2, 100])
def test_masked_states_hold_anything(cuda, hiplib, rows, dtype):
    """NaN and infinities in masked states and behind the last one, whole requests and whole tiles masked, biases of
    fp32's lowest value (all alike: the mean of the values)."""
    import torch
    from tsplat.cross_attention import cross_attention

    queries, keys, heads, D = [rows, rows, rows, rows], [300, 70, 1, 129], 4, 64
    q, k, v, bias, g = _inputs(torch, cuda, queries, keys, heads, 2, D, dtype, 9, extra=40)
    bias[:] = 0
    bias[5], bias[17:160], bias[299] = -INF, -INF, -INF   # whole tiles of the first request
    bias[300:370] = -INF                                  # all of the second
    bias[371:500] = torch.finfo(torch.float32).min        # the fourth
    plan = _plan(torch, cuda, queries, keys, heads, 2, D, dtype)
    want = cross_attention(q, k, v, plan, key_bias=bias)
    assert not want[rows:2 * rows].any()
    k2, v2 = k.clone(), v.clone()
    k2[bias == -INF], v2[bias == -INF] = math.nan, INF
    k2[500:], v2[500:] = -INF, math.nan
    got = cross_attention(q, k2, v2, plan, key_bias=bias)
    assert torch.equal(got[:4 * rows], want[:4 * rows]) and torch.isfinite(got[:4 * rows]).all()
    exact, bound = cross(torch, q[:3 * rows], k[:371], v[:371], queries[:3], keys[:3], bias[:371])
    assert_within(torch, got[:3 * rows].double(), exact, bound, "masked")
    mean, bound = cross(torch, torch.zeros_like(q[3 * rows:4 * rows]), k[371:500], v[371:500], [rows], [129])
    assert_within(torch, got[3 * rows:4 * rows].double(), mean, bound, "lowest")
    # a NaN where a state counts reaches the rows of its request alone
    v2[370] = math.nan
    got = cross_attention(q, k2, v2, plan, key_bias=bias)
    assert torch.isnan(got[2 * rows:3 * rows]).all()
    assert torch.equal(got[:2 * rows], want[:2 * rows]) and torch.equal(got[3 * rows:4 * rows], want[3 * rows:4 * rows])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 90])
def test_far_scores(cuda, hiplib, rows, dtype):
    """Scores that rise from tile to tile by more than a weight's range, and fall again."""
    import torch
    from tsplat.cross_attention import cross_attention

    q, k, v, _, g = _inputs(torch, cuda, [rows], [1500], 2, 2, 64, dtype, 4)
    ramp = torch.cat((torch.linspace(0, 30, 900, device=cuda), torch.linspace(30, -20, 600, device=cuda)))
    q[..., 0] = 8
    k[:, :, 0] = ramp[:, None].to(k.dtype)
    plan = _plan(torch, cuda, [rows], [1500], 2, 2, 64, dtype)
    want, bound = cross(torch, q, k, v, [rows], [1500])
    assert_within(torch, cross_attention(q, k, v, plan).double(), want, bound, "ramp")


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(cuda, hiplib, dtype):
    """Views of fused projections, head-major tensors, odd offsets; rows past the last request and what lies beside the
    result stay as they are."""
    import torch
    from tsplat.cross_attention import cross_attention

    dt = getattr(torch, dtype)
    queries, keys, heads, kv_heads, D = [40, 3], [70, 200], 4, 2, 64
    q, k, v, bias, g = _inputs(torch, cuda, queries, keys, heads, kv_heads, D, dtype, 2, extra=5)
    plan = _plan(torch, cuda, queries, keys, heads, kv_heads, D, dtype)
    want = cross_attention(q, k, v, plan, key_bias=bias)
    assert not want[43:].any() and want.shape == q.shape
    exact, bound = cross(torch, q, k, v, queries, keys, bias)
    flat = torch.randn(48 * heads * 80 + 9, generator=g, device=cuda).to(dt)
    for offset, token, head in ((0, heads * 80, 80), (1, heads * 80, 80), (3, heads * 65, 65), (8, 72, 48 * 72), (2, 70, 48 * 70)):
        q2 = flat.as_strided((48, heads, D), (token, head, 1), offset)
        q2.copy_(q)
        k2 = flat.new_empty(300 * kv_heads * 80 + 9).as_strided((275, kv_heads, D), (kv_heads * 80, 80, 1), offset)
        k2.copy_(k)
        buffer = torch.full((48 * heads * 80 + 9,), 7.0, device=cuda, dtype=dt)
        out = buffer.as_strided((48, heads, D), (token, head, 1), offset)
        assert cross_attention(q2, k2, v, plan, key_bias=bias, out=out) is out
        if dtype == "float32":  # (aligned calls go by pairs of fp16 values, others by bf16 terms)
            assert_within(torch, out[:43].double(), exact[:43], bound[:43], "strides")
        else:
            assert torch.equal(out[:43], want[:43])
        out[:43] = 7.0
        assert bool((buffer == 7).all())


def _outliers(torch, kind, q, k, v):
    """Values that pairs of fp16 under one scale do not hold; the weights of the outlying states are zero or all."""
    if kind == "k early":
        k[3] = -1e6 * q[0, 0].sign()
    elif kind == "k late":
        k[400] = -1e6 * q[0, 0].sign()
    elif kind == "q":
        q[7] *= 1e5
    elif kind == "v early":
        v[2] = 1e12
    elif kind == "v late":
        v[401] = 1e12
    elif kind == "v small":
        v[:, :, 8:16] *= 1e-9
    elif kind == "v steps":
        v[:] *= torch.logspace(-12, 12, len(v), device=v.device)[:, None, None]
    elif kind == "zeros first":
        k[:200], v[:200] = 0.0, 0.0
    elif kind == "all small":
        q *= 1e-15
        k *= 1e-15
        v *= 1e-15
    elif kind == "all large":
        q *= 1e12
        k *= 1e-12
        v *= 1e30
    elif kind == "zero":
        q[:], k[:], v[:] = 0.0, 0.0, 0.0


@pytest.mark.parametrize("kind", ["k early", "k late", "q", "v early", "v late", "v small", "v steps", "zeros first",
                                  "all small", "all large", "zero"])
@pytest.mark.parametrize("D", [64, 128])
def test_values_of_unlike_sizes(cuda, hiplib, kind, D):
    """fp32 accuracy whatever the values' sizes: what one state or feature holds costs no other one anything, and a result
    does not depend on the other requests of the batch."""
    import torch
    from tsplat.cross_attention import cross_attention

    queries, keys = [300, 40, 300], [500, 90, 500]
    q, k, v, bias, g = _inputs(torch, cuda, queries, keys, 2, 2, D, "float32", 12)
    k, v = k.contiguous(), v.contiguous()
    plain = cross_attention(q, k, v, _plan(torch, cuda, queries, keys, 2, 2, D, "float32"))
    _outliers(torch, kind, q[:300], k[:500], v[:500])
    plan = _plan(torch, cuda, queries, keys, 2, 2, D, "float32")
    for b in (None, bias):
        want, bound = cross(torch, q, k, v, queries, keys, b)
        got = cross_attention(q, k, v, plan, key_bias=b)
        if kind == "q":  # scores of 1e5: the bound's first order says nothing for those rows
            rows = torch.arange(640, device=cuda) != 7
            got, want, bound = got[rows], want[rows], bound[rows]
        assert_within(torch, got.double(), want, bound, kind)
        if b is None:
            assert torch.equal(got[-340:], plain[-340:])


def test_offsets_past_32_bits(cuda, hiplib):
    """The last request's states lie behind more than 2^31 values."""
    import torch
    from tsplat.cross_attention import cross_attention

    n, H, D = 70000, 16, 128
    k = torch.empty(n + 50, 17 * H * D, device=cuda, dtype=torch.bfloat16)[:, :H * D].unflatten(1, (H, D))
    g = torch.Generator(device=cuda).manual_seed(6)
    k[n:] = torch.randn(50, H, D, generator=g, device=cuda).to(torch.bfloat16)
    q = torch.randn(2, H, D, generator=g, device=cuda).to(torch.bfloat16)
    plan = _plan(torch, cuda, [0, 2], [n, 50], H, H, D, "bfloat16")
    want, bound = cross(torch, q, k[n:], k[n:], [2], [50])
    assert_within(torch, cross_attention(q, k, k, plan).double(), want, bound, "far")


def test_graphs_streams_and_one_plan(cuda, hiplib):
    """Two captured graphs that share a plan, on two streams, with eager calls between their replays."""
    import torch
    from tsplat.cross_attention import cross_attention

    for queries, keys in (([1, 1], [3000, 50]), ([200, 3], [900, 2000])):
        plan = _plan(torch, cuda, queries, keys, 4, 2, 64, "float32")
        cases = [_inputs(torch, cuda, queries, keys, 4, 2, 64, "float32", seed)[:4] for seed in (1, 2)]
        streams, graphs = [torch.cuda.Stream() for _ in cases], []
        for s, (q, k, v, b) in zip(streams, cases):
            s.wait_stream(torch.cuda.current_stream())
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                y = cross_attention(cross_attention(q, k, v, plan), k, v, plan, key_bias=b)
            graphs.append((graph, y))
        for turn in range(4):
            for q, _, v, _ in cases:
                q.mul_(-0.75), v.mul_(1.25)
            torch.cuda.synchronize()
            for (graph, _), s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
            eager = [cross_attention(cross_attention(q, k, v, plan), k, v, plan, key_bias=b) for q, k, v, b in cases]
            torch.cuda.synchronize()
            for (_, y), e in zip(graphs, eager):
                assert torch.equal(y, e), turn


def test_equal_lengths_agree_with_sdpa(cuda, hiplib):
    """The batch of one length: native_sdpa_f32_ex's result to the rounding of both."""
    import torch
    from tsplat.cross_attention import cross_attention
    from tsplat.native_sdpa_ctypes import native_sdpa_f32_ex

    B, H, Lq, Lk = 2, 4, 300, 150
    q, k, v, _, _ = _inputs(torch, cuda, [Lq] * B, [Lk] * B, H, H, 64, "float32", 8)
    got = cross_attention(q, k, v, _plan(torch, cuda, [Lq] * B, [Lk] * B, H, H, 64, "float32"))
    bhld = [t.unflatten(0, (B, -1)).transpose(1, 2).contiguous() for t in (q, k, v)]
    sdpa = native_sdpa_f32_ex(*bhld, out_layout="blhd").view(B * Lq, H, 64)
    _, bound = cross(torch, q, k, v, [Lq] * B, [Lk] * B)
    assert bool(((got.double() - sdpa.double()).abs() <= 2 * bound).all())


def test_refusals(cuda, hiplib):
    import torch
    from tsplat.cross_attention import CrossPlan, cross_attention

    q, k, v, bias, _ = _inputs(torch, cuda, [5, 2], [9, 30], 4, 2, 64, "float32", 1)
    plan = _plan(torch, cuda, [5, 2], [9, 30], 4, 2, 64, "float32")
    for args, kwargs in (((q[:6], k, v), {}), ((q, k[:38], v), {}), ((q, k, v[:, :1]), {}), ((q.half(), k, v), {}),
                         ((q[..., :32], k, v), {}), ((q.cpu(), k, v), {}), ((q.flatten(), k, v), {}),
                         ((q, k, v), dict(key_bias=bias[:38])), ((q, k, v), dict(key_bias=bias.double())),
                         ((q, k, v), dict(key_bias=bias[None])), ((q, k, v), dict(scale=0.0)),
                         ((q, k, v), dict(scale=math.nan)), ((q, k, v), dict(scale=-1.0)),
                         ((q, k, v), dict(out=q.half())), ((q, k, v), dict(out=q[:6])),
                         ((q.clone().requires_grad_(), k, v), {}),
                         ((q.transpose(1, 2).contiguous().transpose(1, 2), k, v), {})):
        with pytest.raises(ValueError):
            cross_attention(*args, plan, **kwargs)
    with pytest.raises(ValueError):
        cross_attention(q, k, v, None)
    for kwargs in (dict(out=q), dict(out=k.as_strided(q.shape, q.stride()))):
        with pytest.raises(RuntimeError, match="-3"):  # over what is read
            cross_attention(q, k, v, plan, **kwargs)
    with pytest.raises(RuntimeError, match="-3"):  # heads that overlap
        cross_attention(q.as_strided(q.shape, (256, 32, 1)), k, v, plan)
    for args, kwargs in ((([1], [1, 2], 4, 64), {}), (([-1], [1], 4, 64), {}), (([1], [1 << 31], 4, 64), {}),
                         (([1], [1], 4, 129), {}), (([1], [1], 4, 0), {}), (([1], [1], 4, 64), dict(kv_heads=3)),
                         (([1], [1], 4, 64), dict(kv_heads=8)), (([1], [1], 0, 64), {}),
                         (([1], [1], 4, 64), dict(dtype=torch.float64)), (([1], [1], 4, 64), dict(precision="fp8")),
                         (([1], [1], 4, 64), dict(dtype=torch.half, precision="bf16")),
                         (([1], [1], 4, 64), dict(device="cpu")),
                         (([1 << 30, 1 << 30], [1, 1], 4, 64), {}), (([1, 1], [1 << 30, 1 << 30], 4, 64), {})):
        with pytest.raises(ValueError):
            CrossPlan(*args, **{"device": cuda, **kwargs})


def test_handles_used_on_another_stream(cuda, hiplib):
    """A plan and 8-bit rows that are gone before another stream has read them: the allocator keeps their memory."""
    import torch
    from tsplat.cross_attention import cross_attention
    from tsplat.fp8 import fp8_linear, quantize_blocks

    q, k, v, _, g = _inputs(torch, cuda, [300], [2000], 4, 4, 64, "float32", 3)
    w = torch.randn(256, 256, generator=g, device=cuda)
    x = torch.randn(200, 256, generator=g, device=cuda)
    want = cross_attention(q, k, v, _plan(torch, cuda, [300], [2000], 4, 4, 64, "float32"))
    want8 = fp8_linear(x, quantize_blocks(w))
    side = torch.cuda.Stream()
    for _ in range(5):
        plan, weight = _plan(torch, cuda, [300], [2000], 4, 4, 64, "float32"), quantize_blocks(w)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(20):
                got, got8 = cross_attention(q, k, v, plan), fp8_linear(x, weight)
        del plan, weight
        trash = [torch.full((n,), 0x7F, dtype=torch.uint8, device=cuda) for n in (512, 1024, 4096, 70000, 66560) for _ in range(4)]
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(got8, want8)
        del trash
