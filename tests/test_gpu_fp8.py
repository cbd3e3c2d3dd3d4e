"""quantize_blocks and fp8_linear against their definitions in 64 bits: types, odd sizes, strides and alignment, one
row to many, borders of codes and scales, values that are not finite, graphs and streams."""
from __future__ import annotations

import pytest

from _fp8_cases import CUT, STEP, blocks, linear, norm_off, values
from _request_cases import assert_within

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16", "float16"]


def _gen(torch, cuda, seed):
    return torch.Generator(device=cuda).manual_seed(seed)


def _codes_equal(torch, q, x):
    code, e = blocks(torch, x)
    K = x.shape[1]
    code = code.reshape(x.shape[0], -1)
    got = q.codes.float().double()
    assert q.codes.shape == x.shape and q.exponents.shape == e.shape
    assert torch.equal(q.exponents.to(torch.int64), e)
    assert torch.equal(torch.nan_to_num(got, nan=999.0), torch.nan_to_num(code[:, :K], nan=999.0))
    # what lies past K and past the last block
    B = q.blocks
    codes = q._buffer[:x.shape[0] * 128 * B].view(-1, 128 * B)
    exponents = q._buffer[x.shape[0] * 128 * B:].view(x.shape[0], -1)
    assert not codes[:, K:].any() and bool((exponents[:, B:] == 127).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 127), (2, 129), (5, 1000), (33, 512), (64, 4096), (7, 8191),
                                 (1030, 300), (4100, 130), (2, 70001)])
def test_codes(cuda, hiplib, M, K, dtype):
    import torch
    from tsplat.fp8 import quantize_blocks

    print(f"codes M={M} K={K} {dtype}", flush=True)
    g = _gen(torch, cuda, M + K)
    x = torch.randn(M, K, generator=g, device=cuda) * torch.exp(3 * torch.randn(M, 1, generator=g, device=cuda))
    x = x.to(getattr(torch, dtype))
    q = quantize_blocks(x)
    _codes_equal(torch, q, x)
    # (a row whose fp16 values pass the type's range has infinities: NaN on both sides)
    assert torch.equal(torch.nan_to_num(q.dequantize().double(), nan=-7.7), torch.nan_to_num(values(torch, x), nan=-7.7))


def test_borders_of_codes_and_scales(cuda, hiplib):
    """Ties between codes, largest magnitudes next to 448 times a power of two, subnormal codes, the smallest and
    largest fp32 values, blocks of zeros and of negative zeros."""
    import torch
    from tsplat.fp8 import quantize_blocks

    ties = torch.arange(0, 3600, device=cuda, dtype=torch.float32) / 8  # every code up to 448 and what lies between
    rows = []
    for top in (448.0, 448.00003, 447.99997, 464.0, 224.0, 896.0, 1.0):
        for power in (-149, -140, -127, -126, -118, -110, -20, 0, 30, 119):
            row = torch.zeros(1024, device=cuda)
            row[:1000] = ties[torch.arange(1000, device=cuda) * 7 % 3584]
            row[::128] = top
            scaled = row.double() * 2.0 ** power
            rows.append(torch.where(scaled.abs() > 3.4e38, 0.0, scaled).float())
    rows.append(torch.zeros(1024, device=cuda))
    rows.append(-torch.zeros(1024, device=cuda))
    rows.append(torch.full((1024,), 3.4028234663852886e38, device=cuda))
    rows.append(torch.full((1024,), 1e-45, device=cuda))
    x = torch.cat((torch.stack(rows), -torch.stack(rows)))
    _codes_equal(torch, quantize_blocks(x), x)


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite(cuda, hiplib, dtype):
    """They become NaN, and the rest of their block keeps the scale of its finite values."""
    import torch
    from tsplat.fp8 import fp8_linear, quantize_blocks

    x = torch.randn(70, 300, generator=_gen(torch, cuda, 3), device=cuda).to(getattr(torch, dtype))
    x[2, 5], x[3, 200], x[4, 299] = float("inf"), float("-inf"), float("nan")
    x[5, :128] = float("nan")
    _codes_equal(torch, quantize_blocks(x), x)
    w = quantize_blocks(torch.randn(40, 300, generator=_gen(torch, cuda, 4), device=cuda))
    for rows in (x, x[:9]):
        y = fp8_linear(rows, w)
        assert torch.isnan(y[2:6]).all() and torch.isfinite(y[:2]).all() and torch.isfinite(y[6:]).all()


def test_strided_and_unaligned_rows(cuda, hiplib):
    import torch
    from tsplat.fp8 import quantize_blocks

    g = _gen(torch, cuda, 5)
    for dtype in TYPES:
        wide = torch.randn(37, 1201, generator=g, device=cuda).to(getattr(torch, dtype))
        for x in (wide[:, :640], wide[:, 1:513], wide[:, 3:1200], wide[5:6, 2:300], wide[::2, 4:132]):
            _codes_equal(torch, quantize_blocks(x), x)
        x3 = wide[:36, :512].unflatten(0, (4, 9))
        assert torch.equal(quantize_blocks(x3).codes.float(), quantize_blocks(wide[:36, :512]).codes.float())


def _linear_case(torch, cuda, M, K, N, dtype, seed):
    g = _gen(torch, cuda, seed)
    dt = getattr(torch, dtype)
    x = (torch.randn(M, K, generator=g, device=cuda) * (1 + 15 * (torch.rand(K, generator=g, device=cuda) < 0.03))).to(dt)
    w = torch.randn(N, K, generator=g, device=cuda) * K ** -0.5
    bias = torch.randn(N, generator=g, device=cuda)
    residual = torch.randn(M, N, generator=g, device=cuda).to(dt)
    return x, w, bias, residual, g


SIZES = [(1, 64, 64), (1, 1, 1), (2, 129, 17), (5, 1000, 33), (16, 128, 16), (17, 256, 130), (31, 4096, 64),
         (33, 1024, 100), (64, 640, 200), (65, 128, 128), (66, 127, 3), (129, 700, 257), (300, 1000, 1023),
         (777, 1152, 260), (1500, 384, 514), (2100, 136, 1000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear(cuda, hiplib, M, K, N, dtype):
    import torch
    from tsplat.fp8 import fp8_linear, quantize_blocks

    print(f"linear M={M} K={K} N={N} {dtype}", flush=True)
    x, w, bias, residual, g = _linear_case(torch, cuda, M, K, N, dtype, M + N)
    weight = quantize_blocks(w)
    groups = next(d for d in (3, 2, 1) if M % d == 0)
    gate = torch.randn(groups, 2 * N, generator=g, device=cuda)[:, N:]
    for what, args in (("plain", {}), ("bias", dict(bias=bias)), ("gelu", dict(bias=bias, activation="gelu")),
                       ("gated", dict(bias=bias, gate=gate, residual=residual)),
                       ("gate", dict(gate=gate[:1])), ("residual", dict(residual=residual))):
        want, bound = linear(torch, x, w, args.get("bias"), args.get("activation"), args.get("gate"),
                             args.get("residual"), dtype)
        got = fp8_linear(x, weight, **args)
        assert got.dtype is x.dtype
        assert_within(torch, got.double(), want, bound, what)
        if M * N > 1000:
            assert norm_off(torch, got, want) <= STEP[dtype] + (CUT if dtype != "float32" else 2 * K * 2.0 ** -24)
        assert torch.equal(got, fp8_linear(quantize_blocks(x), weight, out_dtype=None if "residual" in args else x.dtype,
                                           **args))
        if "residual" in args:
            inplace = residual.clone()
            assert fp8_linear(x, weight, **{**args, "residual": inplace}, out=inplace) is inplace
            assert torch.equal(inplace, got)


@pytest.mark.parametrize("M", [3, 200])
def test_every_code_times_every_scale(cuda, hiplib, M):
    """Each row and each column pick single values: the products are exact, down to subnormal codes and up to scales
    whose product is as large or small as fp32 holds."""
    import torch
    from tsplat.fp8 import fp8_linear, quantize_blocks

    K, N = 384, 96
    x = torch.zeros(M, K, device=cuda)
    w = torch.zeros(N, K, device=cuda)
    for m in range(M):
        x[m, m * 7 % K] = 1.75 * 2.0 ** (m % 61 - 30) * (-1) ** m
    for n in range(N):
        w[n, ::3] = 1.625 * 2.0 ** (n % 51 - 25)
    got = fp8_linear(x, quantize_blocks(w)).double()
    assert torch.equal(got, x.double() @ w.double().t().contiguous())


def test_linear_strides(cuda, hiplib):
    """Rows of wider tensors, odd offsets, an out that is a column range; what lies beside it stays."""
    import torch
    from tsplat.fp8 import fp8_linear, quantize_blocks

    for dtype in TYPES:
        dt = getattr(torch, dtype)
        for M in (7, 150):
            x, w, bias, _, g = _linear_case(torch, cuda, M, 260, 72, dtype, 11)
            weight = quantize_blocks(w)
            want = fp8_linear(x, weight, bias)
            for lead, skip in ((4, 4), (1, 3), (8, 5)):
                wide_x = torch.randn(M, 300, generator=g, device=cuda).to(dt)
                wide_x[:, lead:lead + 260] = x
                wide = torch.full((M, 72 + lead + skip), 7.0, device=cuda, dtype=dt)
                out = wide[:, lead:lead + 72]
                assert fp8_linear(wide_x[:, lead:lead + 260], weight, bias, out=out) is out
                assert torch.equal(out, want)
                assert bool((wide[:, :lead] == 7).all()) and bool((wide[:, lead + 72:] == 7).all())
        b3 = fp8_linear(x.unflatten(0, (2, -1)), weight, bias)
        assert b3.shape == (2, 75, 72) and torch.equal(b3.flatten(0, 1), want)


def test_graph_and_streams(cuda, hiplib):
    """Two captured graphs and eager calls between their replays, on two streams."""
    import torch
    from tsplat.fp8 import fp8_linear, quantize_blocks

    cases = []
    for seed, M in ((1, 20), (2, 300)):
        x, w, bias, _, _ = _linear_case(torch, cuda, M, 500, 140, "float32", seed)
        cases.append((x, quantize_blocks(w), bias))
    streams = [torch.cuda.Stream() for _ in cases]
    graphs = []
    for s, (x, w, b) in zip(streams, cases):
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            y = fp8_linear(fp8_linear(x, w, b, activation="gelu")[:, :140], quantize_blocks(w.dequantize()[:, :140]))
        graphs.append((graph, y))
    for turn in range(4):
        for x, _, _ in cases:
            x.mul_(-0.75)
        torch.cuda.synchronize()
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        eager = [fp8_linear(fp8_linear(x, w, b, activation="gelu")[:, :140], quantize_blocks(w.dequantize()[:, :140]))
                 for x, w, b in cases]
        torch.cuda.synchronize()
        for (_, y), e in zip(graphs, eager):
            assert torch.equal(y, e), turn


def test_refusals(cuda, hiplib):
    import torch
    from tsplat.fp8 import fp8_linear, quantize_blocks

    x, w, bias, residual, _ = _linear_case(torch, cuda, 70, 130, 40, "float32", 1)
    weight, gate = quantize_blocks(w), torch.ones(2, 40, device=cuda)
    for bad in (x.double(), x.cpu(), x.t(), None, x[:, :0], x.clone().requires_grad_()):
        with pytest.raises(ValueError):
            quantize_blocks(bad)
        with pytest.raises(ValueError):
            fp8_linear(bad, weight)
    for args, kwargs in (((x, w), {}), ((x[:, :129], weight), {}), ((x, weight, bias[:39]), {}),
                         ((x, weight, bias.half()), {}), ((x, weight), dict(activation="relu")),
                         ((x, weight), dict(gate=gate[:, :39])), ((x, weight), dict(gate=torch.ones(3, 40, device=cuda))),
                         ((x, weight), dict(gate=gate.double())), ((x, weight), dict(residual=residual[:69])),
                         ((x, weight), dict(residual=residual, out_dtype=torch.half)),
                         ((x, weight), dict(out=residual[:, :39])), ((x, weight), dict(out_dtype=torch.float64)),
                         ((x, weight), dict(gate=gate[:1].expand(2, -1))), ((x, weight, bias.clone().requires_grad_()), {})):
        with pytest.raises(ValueError):
            fp8_linear(*args, **kwargs)
    with pytest.raises(RuntimeError, match="-3"):
        fp8_linear(x, weight, out=x[:, :40])
    assert quantize_blocks(x[:0]).codes.shape == (0, 130) and fp8_linear(x[:0], weight).shape == (0, 40)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(4200, 136, 4100), (16500, 300, 1030), (1100, 520, 15000), (8192, 1024, 2048)])
def test_linear_of_many_tiles(cuda, hiplib, M, K, N, dtype):
    """More than two of the wide tiles to a CU: ragged bands of rows and runs of columns, each written once."""
    import torch
    from tsplat.fp8 import fp8_linear, quantize_blocks

    print(f"many tiles M={M} K={K} N={N} {dtype}", flush=True)
    x, w, bias, residual, g = _linear_case(torch, cuda, M, K, N, dtype, 21)
    weight, gate = quantize_blocks(w), torch.randn(2, N, generator=g, device=cuda)
    for what, args in (("gelu", dict(bias=bias, activation="gelu")), ("gated", dict(bias=bias, gate=gate, residual=residual))):
        want, bound = linear(torch, x, w, args.get("bias"), args.get("activation"), args.get("gate"), args.get("residual"), dtype)
        assert_within(torch, fp8_linear(x, weight, **args).double(), want, bound, what)
