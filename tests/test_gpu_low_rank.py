"""low_rank_add against its formula in 64 bits: types, ranks, rows of many
adapters, of none, odd sizes, strides, values that only all 24 bits of a
product keep, non-finite values beside the rows, graphs and streams."""
from __future__ import annotations

import pytest

from _request_cases import assert_within, low_rank

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16", "float16"]


def _case(torch, cuda, M, K, N, R, slots, dtype, seed=0, ranks=None):
    from tsplat.adapters import AdapterBank

    g = torch.Generator(device=cuda).manual_seed(seed)
    dt = getattr(torch, dtype)
    ranks = [R] * slots if ranks is None else ranks
    x = torch.randn(M, K, generator=g, device=cuda)
    y = torch.randn(M, N, generator=g, device=cuda)
    down = (torch.randn(slots, R, K, generator=g, device=cuda) / K ** 0.5).to(dt)
    up = torch.randn(slots, N, R, generator=g, device=cuda).to(dt)
    scale = torch.rand(slots, generator=g, device=cuda) + 0.5
    bank = AdapterBank.stack(down, up, scale, ranks)
    adapters = {a: (down[a, :r], up[a, :, :r], float(scale[a])) for a, r in enumerate(ranks) if r > 0}
    return x, y, bank, adapters, g


def _check(torch, x, y, bank, adapters, rows, what):
    from tsplat.adapters import low_rank_add

    got = low_rank_add(y, x, bank, rows)
    want, bound = low_rank(torch, y, x, rows, adapters)
    assert_within(torch, got, want, bound, what)
    bare = torch.tensor([int(a) not in adapters for a in rows.tolist()], device=y.device)
    assert torch.equal(got[bare], y[bare])
    inplace = y.clone()
    assert low_rank_add(inplace, x, bank, rows, out=inplace) is inplace
    assert torch.equal(inplace, got)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N,R", [(1, 64, 64, 16), (1, 1, 1, 1), (2, 1024, 1024, 16), (3, 33, 17, 5), (16, 96, 80, 32),
                                     (17, 100, 50, 33), (33, 257, 130, 48), (63, 513, 65, 64), (64, 1024, 512, 128),
                                     (65, 40, 48, 100), (130, 64, 96, 7), (257, 130, 129, 24), (1030, 192, 160, 17),
                                     (16, 4096, 64, 40), (7, 2050, 6144, 20), (40, 31, 33, 512), (4200, 70, 90, 12), (4300, 200, 72, 100), (4130, 96, 50, 140), (2050, 1100, 70, 90), (2500, 64, 40, 200), (700, 1600, 300, 129),
                                     (9000, 64, 64, 16), (5, 64, 64, 260)])
def test_one_adapter(cuda, hiplib, M, K, N, R, dtype):
    import torch

    print(f"one adapter M={M} K={K} N={N} R={R} {dtype}", flush=True)
    x, y, bank, adapters, _ = _case(torch, cuda, M, K, N, R, 1, dtype, seed=M + R)
    _check(torch, x, y, bank, adapters, torch.zeros(M, dtype=torch.int32, device=cuda), "one")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N,R,slots", [(7000, 64, 40, 20, 5), (6150, 70, 100, 100, 4), (5900, 90, 66, 140, 3),
                                           (9000, 40, 4200, 12, 3), (5000, 40, 6800, 40, 3), (4500, 40, 7500, 70, 1),
                                           (2700, 1100, 90, 130, 6), (300, 1100, 90, 60, 20)])
def test_many_requests_in_every_layout(cuda, hiplib, M, K, N, R, slots, dtype):
    """Requests of ragged lengths that meet inside row tiles, at each count of row, rank and column tiles."""
    import torch

    print(f"layouts M={M} K={K} N={N} R={R} slots={slots} {dtype}", flush=True)
    ranks = [max(1, R - 13 * i) for i in range(slots)]
    x, y, bank, adapters, g = _case(torch, cuda, M, K, N, R, slots, dtype, seed=M, ranks=ranks)
    of_request = torch.randint(-1, slots + 1, (M,), generator=g, device=cuda, dtype=torch.int32)
    starts = torch.rand(M, generator=g, device=cuda) < 0.05
    _check(torch, x, y, bank, adapters, of_request[starts.cumsum(0)], "layouts")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N,R,slots", [(16400, 64, 40, 12, 2), (16400, 70, 33, 25, 2), (16370, 64, 40, 60, 2),
                                           (16390, 40, 50, 100, 2), (24600, 33, 20, 40, 3), (33000, 40, 24, 70, 5),
                                           (16300, 64, 40, 60, 2), (24500, 40, 24, 40, 3), (32700, 40, 24, 70, 5)])
@pytest.mark.parametrize("order", ["requests", "every row another"])
def test_row_tiles_with_and_without_a_border_pass(cuda, hiplib, M, K, N, R, slots, order, dtype):
    """Two row tiles a workgroup and several adapters: so many rows that the workgroup of a border goes through all of
    them by itself, and the last sizes below that."""
    import torch

    print(f"borders M={M} K={K} R={R} slots={slots} {order} {dtype}", flush=True)
    ranks = [max(1, R - 11 * i) for i in range(slots)]
    x, y, bank, adapters, g = _case(torch, cuda, M, K, N, R, slots, dtype, seed=M, ranks=ranks)
    rows = torch.randint(-1, slots + 1, (M,), generator=g, device=cuda, dtype=torch.int32)
    if order == "requests":
        rows = rows[(torch.rand(M, generator=g, device=cuda) < 0.04).cumsum(0)]
    _check(torch, x, y, bank, adapters, rows, "borders")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N,R,slots", [(40, 64, 3000, 33, 64), (130, 96, 3010, 20, 64), (130, 96, 3010, 20, 4),
                                           (70, 64, 9000, 40, 2), (300, 64, 600, 40, 64), (90, 64, 2100, 34, 16)])
def test_column_tiles_by_adapters(cuda, hiplib, M, K, N, R, slots, dtype):
    """Few rows of few and of many adapters, on both sides of where a wave takes more columns."""
    import torch

    print(f"column tiles M={M} N={N} R={R} slots={slots} {dtype}", flush=True)
    ranks = [1 + (R - 1) * (i % 4) // 3 for i in range(slots)]
    x, y, bank, adapters, g = _case(torch, cuda, M, K, N, R, slots, dtype, seed=N + slots, ranks=ranks)
    rows = torch.randint(-1, slots + 1, (M,), generator=g, device=cuda, dtype=torch.int32)
    _check(torch, x, y, bank, adapters, rows, "columns")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N,R,slots", [(64, 256, 192, 16, 64), (64, 256, 192, 32, 5), (300, 128, 160, 24, 7),
                                           (1100, 96, 64, 40, 3), (5000, 96, 80, 16, 9), (9100, 64, 48, 20, 30),
                                           (4600, 130, 70, 128, 6)])
@pytest.mark.parametrize("order", ["requests", "every row another"])
def test_many_adapters(cuda, hiplib, M, K, N, R, slots, order, dtype):
    """Ranks from 0 (an empty slot) to R, rows without an adapter and rows of numbers that are no slots."""
    import torch

    print(f"many adapters M={M} K={K} N={N} R={R} slots={slots} {order} {dtype}", flush=True)
    ranks = [(R * (i % 5)) // 4 if i else R for i in range(slots)]
    x, y, bank, adapters, g = _case(torch, cuda, M, K, N, R, slots, dtype, seed=M, ranks=ranks)
    if order == "requests":
        which = torch.randint(-2, slots + 2, (1 + M // 40,), generator=g, device=cuda)
        rows = which.repeat_interleave(41)[:M].contiguous().to(torch.int32)
        rows = torch.cat([rows, torch.full((M - len(rows),), -1, dtype=torch.int32, device=cuda)])
    else:
        rows = torch.randint(-2, slots + 2, (M,), generator=g, device=cuda, dtype=torch.int32)
    rows[0], rows[-1] = 0, 2 ** 31 - 1
    if M > 3:
        rows[1], rows[2] = -2 ** 31, -1
    _check(torch, x, y, bank, adapters, rows, order)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 40, 2100, 8300])
def test_every_bit_of_a_product(cuda, hiplib, M, dtype):
    """down and up pick single values by powers of two, so that the result is exact: 24 bits of x, and all of an
    adapter's own bits, have to pass through both products."""
    import torch
    from tsplat.adapters import AdapterBank, low_rank_add

    K = N = 48
    R = 20
    g = torch.Generator(device=cuda).manual_seed(M)
    x = torch.randint(-2 ** 24 + 1, 2 ** 24, (M, K), generator=g, device=cuda).float()
    pick = torch.randperm(K, generator=g, device=cuda)[:R]
    down, up = torch.zeros(1, R, K, device=cuda), torch.zeros(1, N, R, device=cuda)
    down[0, torch.arange(R), pick] = 0.25
    up[0, torch.arange(R) * 2, torch.arange(R)] = -2.0
    bank = AdapterBank.stack(down.to(getattr(torch, dtype)), up.to(getattr(torch, dtype)), [1.0])
    rows = torch.zeros(M, dtype=torch.int32, device=cuda)
    got = low_rank_add(torch.zeros(M, N, device=cuda), x, bank, rows)
    want = torch.zeros(M, N, device=cuda)
    want[:, torch.arange(R) * 2] = x[:, pick] * -0.5
    assert torch.equal(got, want)
    # and every bit of the adapter: x and one factor single powers of two
    bits = {"float32": 24, "bfloat16": 8, "float16": 11}[dtype]
    value = torch.randint(2 ** (bits - 1), 2 ** bits, (1, R, K), generator=g, device=cuda).float() / 2 ** (bits - 1)
    value = value.to(getattr(torch, dtype))
    spread = torch.zeros(1, N, R, device=cuda)
    spread[0, torch.arange(R) * 2, torch.arange(R)] = 1.0
    bank = AdapterBank.stack(value, spread.to(getattr(torch, dtype)), [1.0])
    at = torch.randint(0, K, (M,), generator=g, device=cuda)
    one = torch.zeros(M, K, device=cuda)
    one[torch.arange(M), at] = 4.0
    got = low_rank_add(torch.zeros(M, N, device=cuda), one, bank, rows)
    want = torch.zeros(M, N, device=cuda)
    want[:, torch.arange(R) * 2] = value[0, :, at].t().float() * 4.0
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N,R", [(16, 200, 100, 20), (40, 300, 70, 64), (16, 4096, 64, 40), (700, 1600, 300, 129),
                                     (6200, 70, 90, 12), (6300, 200, 72, 30), (6200, 130, 72, 64), (6300, 200, 72, 100),
                                     (6200, 96, 50, 140), (7000, 1100, 70, 90), (9000, 40, 4200, 40)])
def test_every_product_of_terms(cuda, hiplib, M, K, N, R, dtype):
    """One value of x a row, and one of the adapter's second half a column, with all their bits: each output is a product
    of three values, of which every product of their terms counts.  u = 2^-24.

    What the split leaves out of a product is below 2^-22 of it with fp16 weights (4 u) and 2^-21 + 2^-30 with fp32 ones
    (8.1 u); a sum is off by a step, 2 u, of what it holds at most, the whole once and 2^-6 of it before; two such
    products, and u for the scale.  A term that was lost would cost 250 to 1000 u."""
    import torch
    from tsplat.adapters import AdapterBank, low_rank_add

    print(f"terms M={M} K={K} N={N} R={R} {dtype}", flush=True)
    dt, g = getattr(torch, dtype), torch.Generator(device=cuda).manual_seed(M + R)
    # 1 + 2^-7 less a last bit, of 24 and of 11 bits: the largest second terms
    most, most_weight = 1 + 2.0 ** -7 - 2.0 ** -23, {"float32": 1 + 2.0 ** -7 - 2.0 ** -23, "float16": 1 + 7 / 1024}
    value = torch.randn(M, generator=g, device=cuda)
    value[::4] = most
    at = torch.randint(0, K, (M,), generator=g, device=cuda)
    x = torch.zeros(M, K, device=cuda)
    x[torch.arange(M), at] = value
    down = torch.randn(2, R, K, generator=g, device=cuda).to(dt)
    second = torch.randn(2, N, generator=g, device=cuda).to(dt)
    down[:, ::3], second[:, ::2] = most_weight.get(dtype, 1.0), most_weight.get(dtype, 1.0)
    rank_of = torch.arange(N, device=cuda) % R
    up = torch.zeros(2, N, R, dtype=dt, device=cuda)
    up[:, torch.arange(N), rank_of] = second
    scale = torch.tensor([0.7, 1.3], device=cuda)
    rows = torch.randint(0, 2, (M,), generator=g, device=cuda, dtype=torch.int32)
    got = low_rank_add(torch.zeros(M, N, device=cuda), x, AdapterBank.stack(down, up, scale), rows)
    a = rows.long()
    inner = down.double()[a, :, at][:, rank_of]  # [M, N]
    want = (scale.double()[a] * value.double())[:, None] * inner * second.double()[a]
    off = 2 * {"float32": 8.1, "bfloat16": 0.0, "float16": 4.0}[dtype] + 2 * 2.1 + 1
    assert_within(torch, got, want, 1.01 * off * 2.0 ** -24 * want.abs(), "terms")


@pytest.mark.parametrize("dtype", TYPES)
def test_large_and_small_values(cuda, hiplib, dtype):
    """x up to near the end of fp32 and far below 1: nothing on the way overflows or goes to zero that the fp32
    product would keep."""
    import torch

    for size in (1e-30, 1e-12, 1e12, 3e37):
        x, y, bank, adapters, _ = _case(torch, cuda, 50, 64, 40, 16, 1, dtype, seed=3)
        x = (x / x.abs().max() * size).contiguous()
        y = y * size
        adapters = {0: (bank_half(adapters[0][0], 0.25), bank_half(adapters[0][1], 0.0625), 0.5)}
        from tsplat.adapters import AdapterBank

        bank = AdapterBank.stack(adapters[0][0][None], adapters[0][1][None], [0.5])
        _check(torch, x, y, bank, adapters, torch.zeros(50, dtype=torch.int32, device=cuda), f"{size}")


def bank_half(t, f):
    return (t.float() * f).to(t.dtype)


@pytest.mark.parametrize("M", [3, 300, 5000])
def test_values_near_the_smallest(cuda, hiplib, M):
    """A factor counts in steps of 2^-133: x and t are each off by at most that, times the other factor."""
    import torch
    from tsplat.adapters import AdapterBank, low_rank_add

    g = torch.Generator(device=cuda).manual_seed(M)
    for size in (1e-33, 1e-36, 1e-38):
        x = torch.randn(M, 64, generator=g, device=cuda) * size
        down, up = torch.randn(1, 12, 64, generator=g, device=cuda), torch.randn(1, 40, 12, generator=g, device=cuda)
        bank = AdapterBank.stack(down, up, [1.0])
        rows = torch.zeros(M, dtype=torch.int32, device=cuda)
        y = torch.zeros(M, 40, device=cuda)
        want, bound = low_rank(torch, y, x, rows, {0: (down[0], up[0], 1.0)})
        step = 2.0 ** -133
        wide = (down[0].double().abs().sum(1) + 1) @ up[0].double().abs().t().contiguous()
        # (three terms of x and of t, and the smallest fp32 steps of the sums)
        assert_within(torch, low_rank_add(y, x, bank, rows), want, bound + 2 * step * wide, f"{size}")


@pytest.mark.parametrize("M", [1, 2, 40, 300, 5000, 8300])
def test_non_finite_values_stay_in_their_rows(cuda, hiplib, M):
    """NaN and infinities in an adapter, an unloaded slot's memory, scale or a row of x reach only the rows that
    use them."""
    import torch
    from tsplat.adapters import low_rank_add

    print(f"non-finite M={M}", flush=True)
    x, y, bank, adapters, g = _case(torch, cuda, M, 100, 70, 40, 4, "bfloat16", seed=9, ranks=[40, 24, 17, 0])
    rows = torch.randint(-1, 4, (M,), generator=g, device=cuda, dtype=torch.int32)
    rows[0] = 1
    clean = low_rank_add(y, x, bank, rows)
    bank.down[3], bank.up[3], bank.scale[3] = float("nan"), float("inf"), float("nan")
    assert torch.equal(low_rank_add(y, x, bank, rows), clean)
    bank.down[0, :, 1], bank.up[0, 1] = float("inf"), float("nan")
    got = low_rank_add(y, x, bank, rows)
    keep = rows != 0
    assert torch.equal(got[keep], clean[keep])
    bad = torch.rand(M, generator=g, device=cuda) < 0.3
    bad[0] = False
    x2 = torch.where(bad[:, None], torch.tensor(float("nan"), device=cuda), x)
    got = low_rank_add(y, x2, bank, rows)
    same = keep & (~bad | (rows < 0) | (rows == 3))
    assert torch.equal(got[same], clean[same])
    used = bad & (rows > 0) & (rows < 3)
    assert got[used].isnan().all()


@pytest.mark.parametrize("M", [3, 70, 2500, 8200])
def test_strides_and_rows_behind(cuda, hiplib, M):
    """Column ranges of wider rows; what lies beside them and behind the last row is left as it was."""
    import torch
    from tsplat.adapters import low_rank_add

    print(f"strides M={M}", flush=True)
    K, N = 66, 70
    x, y, bank, adapters, g = _case(torch, cuda, M, K, N, 12, 2, "float16", seed=4)
    rows = torch.randint(-1, 2, (M,), generator=g, device=cuda, dtype=torch.int32)
    want = low_rank_add(y, x, bank, rows)
    for pad_x, pad_y, at in ((1, 3, 1), (62, 58, 0), (30, 10, 5)):
        wide_x = torch.full((M + 3, K + pad_x), float("nan"), device=cuda)
        wide_y = torch.full((M + 3, N + pad_y + at), 7.0, device=cuda)
        wide_x[:M, :K], wide_y[:M, at:at + N] = x, y
        vx, vy = wide_x[:M, :K], wide_y[:M, at:at + N]
        assert torch.equal(low_rank_add(vy, vx, bank, rows), want)
        low_rank_add(vy, vx, bank, rows, out=vy)
        assert torch.equal(vy, want)
        wide_y[:M, at:at + N] = 7.0
        assert (wide_y == 7.0).all()
    both = torch.full((M, K + N + 4), 3.0, device=cuda)  # x and y side by side in the same rows
    both[:, :K], both[:, K + 2:K + 2 + N] = x, y
    low_rank_add(both[:, K + 2:K + 2 + N], both[:, :K], bank, rows, out=both[:, K + 2:K + 2 + N])
    assert torch.equal(both[:, K + 2:K + 2 + N], want) and torch.equal(both[:, :K], x)
    assert (both[:, K:K + 2] == 3.0).all() and (both[:, K + 2 + N:] == 3.0).all()
    batch = y[:2 * (M // 2)].view(2, M // 2, N)  # leading dimensions
    got = low_rank_add(batch, x[:2 * (M // 2)].view(2, M // 2, K), bank, rows[:2 * (M // 2)])
    assert got.shape == batch.shape and torch.equal(got.view(-1, N), want[:2 * (M // 2)])


def test_no_rows_and_no_adapters(cuda, hiplib):
    import torch
    from tsplat.adapters import AdapterBank, low_rank_add

    bank = AdapterBank(3, 32, 16, 8, device=cuda)
    none = torch.empty(0, dtype=torch.int32, device=cuda)
    assert low_rank_add(torch.empty(0, 16, device=cuda), torch.empty(0, 32, device=cuda), bank, none).shape == (0, 16)
    for M in (1, 100, 9000):
        y, x = torch.randn(M, 16, device=cuda), torch.randn(M, 32, device=cuda)
        rows = torch.arange(M, dtype=torch.int32, device=cuda) % 5 - 1
        assert torch.equal(low_rank_add(y, x, bank, rows), y)


def test_load_unload(cuda, hiplib):
    """A slot's adapter changes between calls; the calls before keep theirs (one stream)."""
    import torch
    from tsplat.adapters import AdapterBank, low_rank_add

    g = torch.Generator(device=cuda).manual_seed(5)
    bank = AdapterBank(2, 64, 48, 24, torch.bfloat16, cuda)
    x, y = torch.randn(100, 64, generator=g, device=cuda), torch.randn(100, 48, generator=g, device=cuda)
    rows = torch.ones(100, dtype=torch.int32, device=cuda)
    results, wants = [low_rank_add(y, x, bank, rows)], [(y.double(), y.double().abs() + 1)]
    for r in (24, 7, 16):
        down = torch.randn(r, 64, generator=g, device=cuda).bfloat16()
        up = torch.randn(48, r, generator=g, device=cuda).bfloat16()
        bank.load(1, down, up, 0.5)
        results.append(low_rank_add(y, x, bank, rows))
        wants.append(low_rank(torch, y, x, rows, {1: (down, up, 0.5)}))
    bank.unload(1)
    results.append(low_rank_add(y, x, bank, rows))
    for got, (want, bound) in zip(results[:-1], wants):
        assert_within(torch, got, want, bound, "load")
    assert torch.equal(results[0], y) and torch.equal(results[-1], y)


def test_offsets_past_32_bits(cuda, hiplib):
    """Rows whose offsets in x, y and out pass 2^31 values: strided views of few columns."""
    import torch
    from tsplat.adapters import low_rank_add

    M, step = 70, 2 ** 25 + 8   # the last row starts past 2^31 floats
    x, y, bank, adapters, _ = _case(torch, cuda, M, 40, 24, 8, 1, "float32", seed=6)
    rows = torch.zeros(M, dtype=torch.int32, device=cuda)
    want = low_rank_add(y, x, bank, rows)
    big = torch.empty(M * step, device=cuda)
    vx = big.view(M, step)[:, :40]
    vy = big.view(M, step)[:, 64:64 + 24]
    vx.copy_(x)
    vy.copy_(y)
    assert torch.equal(low_rank_add(vy, vx, bank, rows), want)
    low_rank_add(vy, vx, bank, rows, out=vy)
    assert torch.equal(vy, want)


def test_more_rows_than_a_grid_dimension(cuda, hiplib):
    """Row tiles past 65535: the last rows come out as in a call of their own."""
    import torch
    from tsplat.adapters import low_rank_add

    M = 65536 * 16 + 37
    x, y, bank, _, g = _case(torch, cuda, M, 32, 16, 8, 3, "float16", seed=8)
    rows = torch.randint(-1, 4, (M,), generator=g, device=cuda, dtype=torch.int32)
    got = low_rank_add(y, x, bank, rows)
    for a, b in ((0, 5000), (65535 * 16 - 2500, 65535 * 16 + 2500), (M - 5000, M)):  # (rows enough for the same split)
        assert torch.equal(got[a:b], low_rank_add(y[a:b], x[a:b], bank, rows[a:b]))


@pytest.mark.parametrize("M", [2, 600, 8300])
def test_graphs_and_streams(cuda, hiplib, M):
    """Captured without an eager call before, two graphs replayed on two streams at once, and again with eager work
    between: every replay equals the eager result."""
    import torch
    from tsplat.adapters import low_rank_add

    print(f"graphs M={M}", flush=True)
    sets = []
    for seed in (1, 2):
        x, y, bank, _, g = _case(torch, cuda, M, 200, 120, 24, 3, "bfloat16", seed=seed)
        rows = torch.randint(-1, 3, (M,), generator=g, device=cuda, dtype=torch.int32)
        sets.append((x, y, bank, rows, low_rank_add(y, x, bank, rows), torch.empty_like(y)))
    torch.cuda.synchronize(cuda)
    graphs, streams = [], [torch.cuda.Stream(device=cuda) for _ in sets]
    capture = torch.cuda.Stream(device=cuda)
    for x, y, bank, rows, want, out in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=capture):
            low_rank_add(y, x, bank, rows, out=out)
        graphs.append(graph)
    for _ in range(6):
        for s in sets:
            s[5].fill_(float("nan"))
        torch.cuda.synchronize(cuda)
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
                graph.replay()
        eager = low_rank_add(sets[0][1], sets[0][0], sets[0][2], sets[0][3])
        torch.cuda.synchronize(cuda)
        assert torch.equal(eager, sets[0][4])
        for s in sets:
            assert torch.equal(s[5], s[4])


def test_refusals(cuda, hiplib):
    import torch
    from tsplat.adapters import low_rank_add

    x, y, bank, _, _ = _case(torch, cuda, 6, 32, 32, 8, 2, "float32")
    rows = torch.zeros(6, dtype=torch.int32, device=cuda)
    bad = [(y[:5], x, bank, rows, None), (y, x[:, :31], bank, rows, None), (y.double(), x, bank, rows, None),
           (y, x, bank, rows.long(), None), (y, x, bank, rows[:5], None), (y, x, bank, rows.cpu(), None),
           (y.t(), x, bank, rows, None), (y, x, bank, rows, y[:5]), (y, x, bank, rows, torch.empty(6, 31, device=cuda)),
           (y, x.half(), bank, rows, None), (y[:1].expand(6, 32), x, bank, rows, None)]
    for a, b, c, d, out in bad:
        with pytest.raises(ValueError):
            low_rank_add(a, b, c, d, out=out)
    with pytest.raises(ValueError, match="backward"):
        low_rank_add(y.clone().requires_grad_(), x, bank, rows)
    buf = torch.empty(8, 32, device=cuda)
    with pytest.raises(RuntimeError, match="-3"):
        low_rank_add(buf[:6], x, bank, rows, out=buf[1:7])
    with pytest.raises(RuntimeError, match="-3"):
        low_rank_add(y, x, bank, rows, out=x)
    with torch.no_grad():
        low_rank_add(y.clone().requires_grad_(), x, bank, rows)
