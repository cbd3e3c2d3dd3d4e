"""The ragged cross attention's host side, no GPU needed: exported symbols, plans that cover every row and state once, and
what the C entries refuse before any device call."""
from __future__ import annotations

import ctypes
import random
import re
from pathlib import Path

import pytest

HEADER = Path(__file__).resolve().parents[1] / "include" / "tsplat_hip_cross.h"
INTS = 16


@pytest.fixture(scope="module")
def lib():
    from tsplat import load_library

    return load_library()


def test_every_declared_symbol_is_bound(lib):
    from tsplat._lib import CROSS_ABI_VERSION, CROSS_SIGNATURES
    from tsplat.cross_attention import HEADER_INTS

    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    assert set(re.findall(r"\b(tsplat_[a-z0-9_]+)\s*\(", text)) == set(CROSS_SIGNATURES)
    assert lib.tsplat_cross_abi_version() == CROSS_ABI_VERSION
    assert int(re.search(r"TSPLAT_CROSS_HEADER (\d+)", text)[1]) == HEADER_INTS == INTS


def make(lib, queries, keys, heads=4, kv=2, dim=64, dtype=0, precision=0, slack=0):
    n = len(queries)
    ql, kl = ((ctypes.c_int32 * max(1, n))(*x) for x in (queries, keys))
    need = lib.tsplat_cross_plan(ql, kl, n, heads, kv, dim, dtype, precision, None, 0)
    if need < 0:
        return need
    plan = (ctypes.c_int32 * (need + 8))(*[77] * (need + 8))
    got = lib.tsplat_cross_plan(ql, kl, n, heads, kv, dim, dtype, precision, plan, need - slack)
    if slack:
        return got
    assert got == need and list(plan[need:]) == [77] * 8  # (nothing behind the plan)
    return list(plan[:need])


def check(plan, queries, keys, group):
    """Every query row of every request meets every one of its states once, and every part is joined once."""
    items, joins, parts = plan[2:5]
    assert plan[1] == len(plan) == INTS + 8 * (items + joins)
    rows = [plan[INTS + 8 * i:INTS + 8 * i + 8] for i in range(items + joins)]
    seen, part_of = {}, {}
    for token0, row0, n, key0, count, part, _, _ in rows[:items]:
        assert n >= 1 and count >= 0
        seen.setdefault((token0, row0, n), []).append((key0, count, part))
        if part >= 0:
            assert part not in part_of
            part_of[part] = (token0, row0, n)
    assert sorted(part_of) == list(range(parts))
    joined = set()
    for token0, row0, n, first, count, *_ in rows[items:]:
        for part in range(first, first + count):
            assert part_of[part] == (token0, row0, n) and part not in joined
            joined.add(part)
    assert len(joined) == parts
    token0 = key0 = 0
    for nq, nk in zip(queries, keys):
        at = 0
        while at < nq * group:
            n, = {n for t, r, n in seen if (t, r) == (token0, at)}
            ranges = sorted(seen.pop((token0, at, n)))
            assert len(ranges) == 1 or all(p >= 0 for _, _, p in ranges)
            assert len(ranges) > 1 or ranges[0][2] == -1
            here = key0
            for start, count, _ in ranges:
                assert start == here and (count > 0 or nk == 0)
                here += count
            assert here == key0 + nk
            at += n
        assert at == nq * group
        token0, key0 = token0 + nq, key0 + nk
    assert not seen


@pytest.mark.parametrize("dtype,precision", [(0, 0), (0, 1), (0, 2), (1, 0), (2, 0)])
def test_plans_cover_everything_once(lib, dtype, precision):
    rng = random.Random(dtype * 3 + precision)
    cases = [([], []), ([0], [0]), ([1], [0]), ([0], [5]), ([1], [1]), ([1], [100000]), ([16384], [2048]),
             ([1] * 64, [8192] * 64), ([7000, 1], [3, 90000])]
    for _ in range(60):
        n = rng.randint(1, 20)
        top_q, top_k = rng.choice([1, 8, 40, 3000]), rng.choice([1, 50, 300, 20000])
        cases.append(([rng.randint(0, top_q) for _ in range(n)], [rng.randint(0, top_k) for _ in range(n)]))
    for queries, keys in cases:
        for heads, kv, dim in ((1, 1, 64), (4, 2, 128), (24, 3, 72)):
            plan = make(lib, queries, keys, heads, kv, dim, dtype, precision)
            check(plan, queries, keys, heads // kv)
            assert plan[5:7] == [sum(queries), sum(keys)]
            assert lib.tsplat_cross_scratch_bytes((ctypes.c_int32 * INTS)(*plan[:INTS])) >= 0


@pytest.mark.parametrize("change", [dict(queries=[-1]), dict(keys=[-1]), dict(heads=0), dict(kv=0), dict(kv=3),
                                    dict(dim=0), dict(dim=129), dict(dtype=3), dict(dtype=-1), dict(precision=3),
                                    dict(precision=-1), dict(dtype=1, precision=1), dict(heads=1 << 16, kv=1),
                                    dict(queries=[2 ** 31 - 1]), dict(keys=[2 ** 31 - 1])])
def test_plan_refusals(lib, change):
    args = {"queries": [3], "keys": [5], **change}
    assert make(lib, **args) == -2


def test_plan_of_more_workgroups_than_a_launch_has(lib):
    n = 1 << 18
    assert len(make(lib, [1] * n, [1] * n, heads=16, kv=16)) == INTS + 8 * n
    assert make(lib, [1] * n, [1] * n, heads=128, kv=128) == -2


def test_plan_of_too_little_room_or_no_lengths(lib):
    assert make(lib, [3, 700], [5, 9], slack=1) == -3
    assert lib.tsplat_cross_plan(None, None, 1, 4, 2, 64, 0, 0, None, 0) == -1
    assert lib.tsplat_cross_plan(None, None, -1, 4, 2, 64, 0, 0, None, 0) == -2


P = [0x10000000 * (i + 1) for i in range(8)]  # never read: every call below is refused before


def _call(lib, q=P[0], qt=256, qh=64, k=P[1], kt=256, kh=64, v=P[2], vt=256, vh=64, bias=None, scale=0.125, out=P[3],
          ot=256, oh=64, header=None, plan=P[4], scratch=P[5], size=1 << 40, queries=(5, 60), keys=(9, 3000), **header_at):
    ints = make(lib, list(queries), list(keys), 4, 2)[:INTS]
    for at, value in header_at.items():
        ints[int(at[1:])] = value
    h = (ctypes.c_int32 * INTS)(*ints)
    return lib.tsplat_cross_attention_async(q, qt, qh, k, kt, kh, v, vt, vh, bias, scale, out, ot, oh,
                                            h if header is None else header, plan, scratch, size, None)


@pytest.mark.parametrize("change,status", [
    (dict(header=0), -1), (dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(out=None), -1),
    (dict(plan=None), -1),
    (dict(scale=0.0), -2), (dict(scale=float("nan")), -2), (dict(scale=float("inf")), -2), (dict(scale=-1.0), -2),
    (dict(h0=1), -2), (dict(h1=5), -2), (dict(h2=-1), -2), (dict(h3=1000000), -2), (dict(h4=1 << 30), -2),
    (dict(h5=-1), -2), (dict(h6=-1), -2), (dict(h7=5), -2), (dict(h8=0), -2), (dict(h9=129), -2), (dict(h9=0), -2),
    (dict(h10=3), -2), (dict(h11=0), -2), (dict(h11=4), -2), (dict(h10=1), -2),
    (dict(qt=255), -3), (dict(qh=63), -3), (dict(kt=127, kh=64), -3), (dict(kh=63), -3), (dict(vt=127), -3), (dict(vh=0), -3),
    (dict(ot=255), -3), (dict(oh=63), -3), (dict(qt=1 << 60), -3), (dict(qt=-256), -3),
    (dict(out=P[0]), -3), (dict(out=P[1]), -3), (dict(out=P[2] + 4), -3), (dict(out=P[4]), -3),
    (dict(bias=P[3] + 64), -3), (dict(scratch=P[0]), -3), (dict(scratch=P[1]), -3), (dict(scratch=P[3]), -3),
    (dict(scratch=P[4]), -3), (dict(bias=P[5]), -3),
    (dict(scratch=None), -5), (dict(size=16), -5),
    (dict(q=P[0] + 2), -4), (dict(k=P[1] + 1), -4), (dict(v=P[2] + 2), -4), (dict(out=P[3] + 1), -4),
    (dict(bias=P[6] + 2), -4), (dict(plan=P[4] + 2), -4), (dict(scratch=P[5] + 8), -4),
    ({}, -6), (dict(bias=P[6]), -6)])
def test_refusals(lib, change, status):
    if change == dict(header=0):
        assert lib.tsplat_cross_attention_async(*[P[0], 256, 64] * 3, None, 0.125, P[3], 256, 64, None, P[4], None, 0,
                                                None) == status
        return
    got = _call(lib, **change)
    assert got == status or (status == -6 and got == -7)


def test_nothing_to_do(lib):
    assert _call(lib, queries=(0, 0), keys=(5, 9), q=None, out=None) == 0


def test_scratch_of_no_header(lib):
    assert lib.tsplat_cross_scratch_bytes(None) == 0
    assert lib.tsplat_cross_scratch_bytes((ctypes.c_int32 * INTS)()) == 0
