"""The 8-bit rows' and products' host side, no GPU needed: exported symbols, and what the C entries refuse before any
device call."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

HEADER = Path(__file__).resolve().parents[1] / "include" / "tsplat_hip_fp8.h"
P = [0x10000000 * (i + 1) for i in range(12)]  # never read: every call below is refused before
BIG = 2 ** 31 - 1


@pytest.fixture(scope="module")
def lib():
    from tsplat import load_library

    return load_library()


def test_every_declared_symbol_is_bound(lib):
    from tsplat._lib import FP8_ABI_VERSION, FP8_SIGNATURES

    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    assert set(re.findall(r"\b(tsplat_[a-z0-9_]+)\s*\(", text)) == set(FP8_SIGNATURES)
    assert lib.tsplat_fp8_abi_version() == FP8_ABI_VERSION


@pytest.mark.parametrize("name,text", [("FP8_ABI_VERSION", "8-bit products"), ("CROSS_ABI_VERSION", "cross attention")])
def test_another_version_is_refused(lib, monkeypatch, name, text):
    from tsplat import _lib

    monkeypatch.setattr(_lib, name, getattr(_lib, name) + 1)
    monkeypatch.setattr(_lib, "_CACHE", {})
    with pytest.raises(RuntimeError, match=text):
        _lib.load_library()


def _quantize(lib, x=P[0], dtype=0, stride=200, rows=6, K=200, codes=P[1], exps=P[2]):
    return lib.tsplat_fp8_quantize_async(x, dtype, stride, rows, K, codes, exps, None)


@pytest.mark.parametrize("change,status", [
    (dict(x=None), -1), (dict(codes=None), -1), (dict(exps=None), -1),
    (dict(dtype=3), -2), (dict(dtype=-1), -2), (dict(rows=0), -2), (dict(rows=-1), -2), (dict(rows=(1 << 27) + 1), -2),
    (dict(K=0), -2), (dict(K=(1 << 20) + 1), -2),
    (dict(stride=199), -3), (dict(stride=-200), -3), (dict(stride=1 << 62), -3),
    (dict(codes=P[0]), -3), (dict(codes=P[0] + 4 * 200 * 6 - 16), -3), (dict(codes=P[0] - 256 * 6 + 16), -3),
    (dict(exps=P[0]), -3), (dict(exps=P[1]), -3), (dict(exps=P[1] + 256 * 6 - 4), -3), (dict(exps=P[1] - 20), -3),
    (dict(x=P[0] + 2), -4), (dict(x=P[0] + 1, dtype=1), -4), (dict(codes=P[1] + 8), -4), (dict(exps=P[2] + 2), -4),
    ({}, -6), (dict(exps=P[2] + 4), -6), (dict(x=P[0] + 2, dtype=2), -6), (dict(codes=P[0] - 256 * 6), -6)])
def test_quantize_refusals(lib, change, status):
    got = _quantize(lib, **change)
    assert got == status or (status == -6 and got == -7)


def _linear(lib, x=P[0], xt=0, xs=200, xc=None, xe=None, wc=P[1], we=P[2], bias=P[3], act=0, gate=P[4], gs=300, per=50,
            residual=P[5], rs=300, out=P[6], ot=0, os=300, M=100, K=200, N=300, scratch=P[7], size=1 << 40):
    return lib.tsplat_fp8_linear_async(x, xt, xs, xc, xe, wc, we, bias, act, gate, gs, per, residual, rs, out, ot, os, M, K,
                                       N, scratch, size, None)


ROWS = dict(x=None, xc=P[8], xe=P[9])


@pytest.mark.parametrize("change,status", [
    (dict(x=None), -1), (dict(x=None, xc=P[8]), -1), (dict(x=None, xe=P[9]), -1), (dict(wc=None), -1),
    (dict(we=None), -1), (dict(out=None), -1),
    (dict(M=0), -2), (dict(K=0), -2), (dict(N=0), -2), (dict(M=BIG), -2), (dict(K=BIG), -2), (dict(N=BIG), -2),
    (dict(xt=3), -2), (dict(ot=-1), -2), (dict(act=2), -2),
    (dict(xs=199), -3), (dict(os=299), -3), (dict(rs=299), -3), (dict(gs=299), -3), (dict(per=0), -3),
    (dict(gs=-300), -3), (dict(os=1 << 60), -3),
    (dict(out=P[0]), -3), (dict(out=P[1]), -3), (dict(out=P[2]), -3), (dict(out=P[3]), -3), (dict(out=P[4]), -3),
    (dict(out=P[5] + 4), -3), (dict(out=P[5], os=301), -3), (dict(out=P[8], **ROWS), -3), (dict(out=P[9], **ROWS), -3),
    (dict(scratch=P[0]), -3), (dict(scratch=P[1]), -3), (dict(scratch=P[3]), -3), (dict(scratch=P[4]), -3),
    (dict(scratch=P[5]), -3), (dict(scratch=P[6]), -3), (dict(scratch=P[2]), -3),
    (dict(scratch=None), -5), (dict(size=100), -5),
    (dict(x=P[0] + 2), -4), (dict(out=P[6] + 2), -4), (dict(out=P[6] + 1, residual=None, ot=1), -4), (dict(residual=P[5] + 1), -4),
    (dict(bias=P[3] + 2), -4), (dict(gate=P[4] + 1), -4), (dict(wc=P[1] + 8), -4), (dict(we=P[2] + 2), -4),
    (dict(scratch=P[7] + 8), -4), (dict(x=None, xc=P[8] + 4, xe=P[9]), -4), (dict(x=None, xc=P[8], xe=P[9] + 1), -4),
    ({}, -6), (ROWS, -6), (dict(ROWS, scratch=None), -6), (dict(M=64, scratch=None), -6), (dict(out=P[5]), -6),
    (dict(gate=None, residual=None, bias=None), -6), (dict(gs=0, per=1), -6)])
def test_linear_refusals(lib, change, status):
    got = _linear(lib, **change)
    assert got == status or (status == -6 and got == -7)


def test_scratch(lib):
    size = lib.tsplat_fp8_linear_scratch_bytes
    assert size(65, 200, 300, 1) == 65 * (256 + 4) // 16 * 16 + 16 * (65 * 260 % 16 > 0)
    assert size(64, 200, 300, 1) == 0 == size(65, 200, 300, 0)
    for bad in ((0, 200, 300), (BIG, 200, 300), (65, 0, 300), (65, BIG, 300), (65, 200, 0), (65, 200, BIG), (-1, 1, 1)):
        assert size(*bad, 1) == 0
