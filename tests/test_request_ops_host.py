"""The request operators' host side, no GPU needed: exported symbols, the
layout of an adapter bank, positions' plans, and what the C entries and the
wrappers refuse before any device call."""
from __future__ import annotations

import math
import re
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "tsplat_hip_requests.h"


@pytest.fixture(scope="module")
def lib():
    from tsplat import load_library

    return load_library()


def test_every_declared_symbol_is_bound(lib):
    from tsplat._lib import REQUEST_SIGNATURES, REQUESTS_ABI_VERSION

    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    declared = set(re.findall(r"\b(tsplat_[a-z0-9_]+)\s*\(", text))
    assert declared == set(REQUEST_SIGNATURES)
    assert lib.tsplat_requests_abi_version() == REQUESTS_ABI_VERSION


def test_another_version_is_refused(lib, monkeypatch):
    from tsplat import _lib

    monkeypatch.setattr(_lib, "REQUESTS_ABI_VERSION", _lib.REQUESTS_ABI_VERSION + 1)
    monkeypatch.setattr(_lib, "_CACHE", {})
    with pytest.raises(RuntimeError, match="request operators"):
        _lib.load_library()


P = [0x100000 * (i + 1) for i in range(16)]  # never read: every call below is refused before


def _low_rank(lib, y=P[0], ys=64, x=P[1], xs=64, rows=P[2], down=P[3], up=P[4], scale=P[5], rank=P[6], out=P[7],
              os=64, M=4, K=64, N=64, slots=2, R=16, dtype=1, scratch=P[8], size=1 << 40):
    return lib.tsplat_low_rank_add_async(y, ys, x, xs, rows, down, up, scale, rank, out, os, M, K, N, slots, R,
                                         dtype, scratch, size, None)


@pytest.mark.parametrize("change,status", [
    (dict(y=None), -1), (dict(x=None), -1), (dict(rows=None), -1), (dict(down=None), -1), (dict(up=None), -1),
    (dict(scale=None), -1), (dict(rank=None), -1), (dict(out=None), -1),
    (dict(M=0), -2), (dict(K=0), -2), (dict(N=0), -2), (dict(slots=0), -2), (dict(R=0), -2), (dict(R=513), -2),
    (dict(dtype=3), -2), (dict(M=-1), -2), (dict(slots=(1 << 20) + 1), -2), (dict(K=(1 << 20) + 1), -2), (dict(N=(1 << 20) + 1), -2), (dict(M=(1 << 27) + 1), -2),
    (dict(ys=63), -3), (dict(xs=63), -3), (dict(os=63), -3), (dict(ys=1 << 60), -3),
    (dict(out=P[0] + 64), -3),                 # over y, but not y itself
    (dict(out=P[0], os=65), -3),               # y at another stride
    (dict(out=P[1]), -3), (dict(out=P[1] + 4 * 32, xs=128, os=128), -3),  # over x
    (dict(down=P[3] + 8), -4), (dict(up=P[4] + 2), -4), (dict(x=P[1] + 2), -4), (dict(rows=P[2] + 1), -4),
])
def test_low_rank_refusals(lib, change, status):
    assert _low_rank(lib, **change) == status


def test_low_rank_scratch(lib):
    sizes = (300, 64, 64, 2, 16, 1)
    need = lib.tsplat_low_rank_scratch_bytes(*sizes)
    assert need >= 0
    if need:
        assert _low_rank(lib, M=300, scratch=None) == -5
        assert _low_rank(lib, M=300, size=need - 1) == -5
        assert _low_rank(lib, M=300, scratch=P[8] + 4) == -4
    assert lib.tsplat_low_rank_scratch_bytes(0, 64, 64, 2, 16, 1) == 0


@pytest.mark.parametrize("change", [
    dict(rows=P[7]), dict(rows=P[7] - 4 * 299), dict(rows=P[7] + 4 * (300 * 64 - 1)), dict(scale=P[7]),
    dict(scale=P[7] - 4), dict(rank=P[7] + 64), dict(down=P[7]), dict(down=P[7] - 4080), dict(up=P[7] - 8176),
    dict(rows=P[8]), dict(scale=P[8]), dict(rank=P[8] + 4), dict(down=P[8]), dict(up=P[8]),
    dict(x=P[8]), dict(y=P[8]), dict(out=P[8]), dict(y=P[8], out=P[8]), dict(scratch=P[1] + 4 * 300 * 64 - 16)])
def test_low_rank_memory_that_is_written_over_what_is_read(lib, change):
    """out (300 rows) or scratch over one value of the rows, an adapter (2 slots: down 4096 bytes, up 8192), scale, rank;
    scratch over x, y and out."""
    assert _low_rank(lib, M=300, **change) == -3


@pytest.mark.parametrize("change", [dict(rows=P[7] - 4 * 300), dict(rows=P[7] + 4 * 300 * 64), dict(scale=P[7] - 8),
                                    dict(down=P[7] - 4096), dict(up=P[7] - 8192), dict(scratch=P[1] + 4 * 300 * 64),
                                    dict(M=16, scratch=P[7]), dict(out=P[0])])
def test_low_rank_memory_beside_what_is_read(lib, change):
    """Up to the edges (and scratch that the call does not use): refused only as memory that is none of a device."""
    assert _low_rank(lib, **{"M": 300, **change}) in (-6, -7)


@pytest.mark.parametrize("at,value", [(0, 2 ** 31 - 1), (0, (1 << 27) + 1), (0, -1), (1, 2 ** 31 - 1),
                                      (1, (1 << 20) + 1), (1, 0), (2, 2 ** 31 - 1), (2, (1 << 20) + 1), (2, -5),
                                      (3, (1 << 20) + 1), (3, 0), (4, 513), (4, 0), (5, 3), (5, -1)])
def test_no_scratch_for_sizes_that_are_refused(lib, at, value):
    sizes = [300, 64, 64, 2, 16, 1]
    assert lib.tsplat_low_rank_scratch_bytes(*sizes) > 0
    sizes[at] = value
    assert lib.tsplat_low_rank_scratch_bytes(*sizes) == 0


def _norm(lib, x=P[0], xs=32, h=P[1], hs=32, out=P[2], os=32, normed=P[3], ns=32, rows=4, cols=32, c=1.0, gate=None,
          gs=0, post=0, pw=None, pb=None, pe=1e-6, pre=1, w=None, b=None, e=1e-6, scale=None, shift=None, ms=0, per=2):
    return lib.tsplat_residual_norm_async(x, xs, h, hs, out, os, normed, ns, rows, cols, c, gate, gs, post, pw, pb,
                                          pe, pre, w, b, e, scale, shift, ms, per, None)


@pytest.mark.parametrize("change,status", [
    (dict(x=None), -1), (dict(h=None), -1), (dict(out=None), -1), (dict(normed=None), -1),
    (dict(rows=0), -2), (dict(rows=1 << 31), -2), (dict(cols=0), -2), (dict(e=-1.0), -2), (dict(pe=float("nan")), -2),
    (dict(pre=0), -2), (dict(pre=3), -2), (dict(post=3), -2),
    (dict(xs=31), -3), (dict(hs=31), -3), (dict(os=31), -3), (dict(ns=31), -3),
    (dict(scale=P[5], ms=32), -3), (dict(shift=P[5], ms=32), -3), (dict(pw=P[5]), -3),
    (dict(gate=P[5], gs=31), -3), (dict(gate=P[2], gs=32, per=(1 << 63) - 1), -3), (dict(gate=P[5], gs=32, per=0), -3),
    (dict(out=P[0] + 4), -3), (dict(out=P[1]), -3), (dict(normed=P[0]), -3), (dict(normed=P[2]), -3),
    (dict(normed=P[1] + 4), -3), (dict(gate=P[2], gs=32), -3), (dict(scale=P[3], shift=P[5], ms=32), -3),
    (dict(x=P[0] + 1), -4),
])
def test_residual_norm_refusals(lib, change, status):
    assert _norm(lib, **change) == status


def _rope(lib, x=P[0], ps=0, sb=0, sl=128, sh=64, parts=1, g0=None, g1=None, o0=P[1], o1=None, o2=None, pos=P[4],
          ptype=0, pb=1, axes=2, turns=P[5], axis=P[6], inter=1, eps=1e-12, B=1, L=4, H=2, D=64, bhld=1):
    return lib.tsplat_rope_axes_async(x, ps, sb, sl, sh, parts, g0, g1, o0, o1, o2, pos, ptype, pb, axes, turns, axis,
                                      inter, eps, B, L, H, D, bhld, None)


@pytest.mark.parametrize("change,status", [
    (dict(x=None), -1), (dict(o0=None), -1), (dict(pos=None), -1), (dict(turns=None), -1), (dict(axis=None), -1),
    (dict(parts=2, ps=64), -1), (dict(parts=3, ps=64, o1=P[2]), -1),
    (dict(parts=0), -2), (dict(parts=4), -2), (dict(B=0), -2), (dict(L=0), -2), (dict(H=0), -2), (dict(D=63), -2),
    (dict(D=514), -2), (dict(H=(1 << 16) + 1), -2), (dict(axes=0), -2), (dict(axes=9), -2), (dict(ptype=2), -2), (dict(eps=-1.0), -2),
    (dict(B=1 << 16, L=1 << 16, sb=64), -2),
    (dict(pb=2), -3), (dict(sh=63), -3), (dict(sl=-128), -3), (dict(sl=1 << 62), -3), (dict(B=2, sb=0), -3),
    (dict(o0=P[0]), -3), (dict(parts=2, ps=64, o1=P[1] + 4), -3),
    (dict(x=P[0] + 2), -4), (dict(turns=P[5] + 4), -4), (dict(g0=P[3] + 1), -4),
])
def test_rope_refusals(lib, change, status):
    assert _rope(lib, **change) == status


@pytest.mark.parametrize("change", [
    dict(g0=P[1] + 2044), dict(g0=P[1] - 508), dict(pos=P[1]), dict(pos=P[1] - 28), dict(turns=P[1] + 2040),
    dict(turns=P[1] - 248), dict(axis=P[1] + 1024), dict(axis=P[1] - 124),
    dict(parts=2, ps=512, o1=P[2], g1=P[2]), dict(parts=2, ps=512, o1=P[2], pos=P[2] + 2044),
    dict(parts=3, ps=512, o1=P[2], o2=P[3], g0=P[3] - 508)])
def test_rope_outputs_over_what_is_read(lib, change):
    """An output of 2048 bytes over one value of a gamma (512 bytes), the positions (32), turns (256) or axis (128)."""
    assert _rope(lib, **change) == -3


@pytest.mark.parametrize("change", [dict(g0=P[1] + 2048), dict(g0=P[1] - 512), dict(pos=P[1] - 32),
                                    dict(turns=P[1] - 256), dict(axis=P[1] - 128), dict(g1=P[1])])
def test_rope_outputs_beside_what_is_read(lib, change):
    """Up to its edges an output is taken (a gamma of a part that the call lacks is not read): only the memory itself,
    which is none of a device, is refused."""
    assert _rope(lib, **change) in (-6, -7)


def test_host_memory_is_refused(lib):
    """Pointers that are no device memory are -6 (or a failed query of them), never a launch."""
    assert _low_rank(lib) in (-6, -7)
    assert _norm(lib) in (-6, -7)
    assert _rope(lib) in (-6, -7)


def test_wrappers_refuse_cpu_tensors():
    import torch
    from tsplat.adapters import AdapterBank, low_rank_add
    from tsplat.block_ops import residual_norm
    from tsplat.qkv import RopeAxes, qkv_rope_axes, rope_axes

    bank = AdapterBank(2, 8, 8, 4, device="cpu")
    t = torch.zeros(3, 8)
    with pytest.raises(ValueError, match="GPU"):
        low_rank_add(t, t.clone(), bank, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="AdapterBank"):
        low_rank_add(t, t.clone(), None, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU"):
        residual_norm(t, t.clone())
    with pytest.raises(ValueError, match="norm is"):
        residual_norm(t, t.clone(), norm=None)
    rope = RopeAxes(8, [2, 2], device="cpu")
    with pytest.raises(ValueError, match="GPU"):
        rope_axes(torch.zeros(1, 3, 1, 8), torch.zeros(3, 2, dtype=torch.int32), rope)
    with pytest.raises(ValueError, match="GPU"):
        qkv_rope_axes(torch.zeros(3, 24), torch.zeros(3, 2, dtype=torch.int32), rope, None, None, 1, 3, 1)


def _value(bank, half, slot, row, col):
    at = (col % 32 // 8, row % 16, col % 8)
    tile = half[slot, row // 16, col // 32]
    return sum(tile[(i, *at)].float() for i in range(3)) if tile.dim() == 4 else tile[at]


@pytest.mark.parametrize("K,N,R,dtype", [(64, 32, 16, "float32"), (33, 17, 5, "bfloat16"), (7, 100, 40, "float16")])
def test_bank_layout(K, N, R, dtype):
    """Every value is where the header says, zeros elsewhere; load, stack and unload agree, and a smaller adapter
    leaves nothing of a larger one behind."""
    import torch
    from tsplat.adapters import AdapterBank

    dt = getattr(torch, dtype)
    g = torch.Generator().manual_seed(1)
    down, up = torch.randn(2, R, K, generator=g).to(dt), torch.randn(2, N, R, generator=g).to(dt)
    small = max(1, R // 2)
    stacked = AdapterBank.stack(down, up, torch.tensor([0.5, 2.0]), [R, small])
    bank = AdapterBank(2, K, N, R, dt, device="cpu")
    bank.load(0, down[0], up[0], 0.5)
    bank.load(1, down[0], up[0], 1.0)
    bank.load(1, down[1, :small], up[1, :, :small], 2.0)
    for key in ("down", "up", "scale", "rank"):
        assert torch.equal(getattr(bank, key), getattr(stacked, key)), key
    for slot, rank in ((0, R), (1, small)):
        for r, k in [(0, 0), (rank - 1, K - 1), (rank // 2, K // 2)]:
            assert _value(bank, bank.down, slot, r, k) == down[slot, r, k]
        for n, r in [(0, 0), (N - 1, rank - 1), (N // 2, rank // 2)]:
            assert _value(bank, bank.up, slot, n, r) == up[slot, n, r]
        planes = 3 if dtype == "float32" else 1
        assert int((bank.down[slot] != 0).sum()) <= planes * rank * K
        assert int((bank.up[slot] != 0).sum()) <= planes * rank * N
    bank.unload(0)
    assert bank.rank.tolist() == [0, small]


def test_bank_refusals():
    import torch
    from tsplat.adapters import AdapterBank, adapter_rows

    bank = AdapterBank(2, 8, 6, 4, device="cpu")
    for slot, down, up in [(2, (4, 8), (6, 4)), (-1, (4, 8), (6, 4)), (0, (5, 8), (6, 5)), (0, (0, 8), (6, 0)),
                           (0, (4, 7), (6, 4)), (0, (4, 8), (7, 4)), (0, (4, 8), (6, 3))]:
        with pytest.raises(ValueError):
            bank.load(slot, torch.zeros(down), torch.zeros(up))
    with pytest.raises(ValueError):
        AdapterBank(2, 8, 6, 513, device="cpu")
    for sizes in ((0, 8, 6, 4), (2, 0, 6, 4), (2, 8, 0, 4), (2, 8, 6, 0), ((1 << 20) + 1, 8, 6, 4),
                  (2, (1 << 20) + 1, 6, 4), (2, 8, (1 << 20) + 1, 4)):
        with pytest.raises(ValueError):
            AdapterBank(*sizes, device="meta")
    with pytest.raises(ValueError):
        AdapterBank(2, 8, 6, 4, torch.float64, device="cpu")
    with pytest.raises(ValueError):
        AdapterBank.stack(torch.zeros(2, 4, 8), torch.zeros(2, 6, 4), [1.0, 1.0], [4, 5])
    with pytest.raises(ValueError):
        AdapterBank.stack(torch.zeros(2, 4, 8), torch.zeros(2, 6, 4), [1.0])
    assert adapter_rows([2, 0, 3], [5, 1, -1], "cpu").tolist() == [5, 5, -1, -1, -1]
    assert adapter_rows([], [], "cpu").tolist() == []
    with pytest.raises(ValueError):
        adapter_rows([1], [1, 2], "cpu")


def test_rope_plan():
    import torch
    from tsplat.qkv import RopeAxes

    own = RopeAxes(12, [1, 2, 3], 100.0, device="cpu")
    assert own.axis.tolist() == [0, 1, 1, 2, 2, 2] and own.axes == 3
    want = [1, 1, 100 ** -0.5, 1, 100 ** (-1 / 3), 100 ** (-2 / 3)]
    assert torch.allclose(own.turns * 2 * math.pi, torch.tensor(want, dtype=torch.float64), rtol=1e-15, atol=0)
    shared = RopeAxes(12, [2, 4], 100.0, shared=True, device="cpu")
    want = [100 ** (-p / 6) for p in range(6)]
    assert torch.allclose(shared.turns * 2 * math.pi, torch.tensor(want, dtype=torch.float64), rtol=1e-15, atol=0)
    assert RopeAxes(8, [0, 4], device="cpu").axis.tolist() == [1] * 4
    for bad in [(7, [3]), (8, [3]), (8, [5, -1]), (8, []), (514, [257]), (0, [0]), (20, [1] * 9 + [1])]:
        with pytest.raises(ValueError):
            RopeAxes(*bad, device="cpu")
    with pytest.raises(ValueError):
        RopeAxes(8, [4], 0.0, device="cpu")


def test_a_library_is_found_by_what_its_name_means_now(lib, monkeypatch, tmp_path):
    """The library of no name is found again at once; a name that is given is looked up in every call."""
    import shutil

    from tsplat import load_library
    from tsplat._lib import DEFAULT_LIBRARY

    monkeypatch.delenv("TSPLAT_HIP_LIBRARY", raising=False)
    monkeypatch.chdir(tmp_path)
    default = load_library()
    assert load_library() is default and load_library(DEFAULT_LIBRARY) is default
    with pytest.raises(FileNotFoundError):
        load_library("")
    other = tmp_path / "other.so"
    shutil.copy(DEFAULT_LIBRARY, other)
    link = tmp_path / "link.so"
    for target in (DEFAULT_LIBRARY, other):
        link.unlink(missing_ok=True)
        link.symlink_to(target)
        for _ in range(3):
            assert load_library(str(link)) is load_library(target)
            monkeypatch.setenv("TSPLAT_HIP_LIBRARY", str(link))
            assert load_library() is load_library(target)
            monkeypatch.delenv("TSPLAT_HIP_LIBRARY")
    assert load_library(str(link)) is not default
    link.unlink()
    with pytest.raises(FileNotFoundError):
        load_library(str(link))
    assert load_library() is default


def test_tangents_are_refused_like_gradients():
    """A tensor with a forward-mode tangent has none afterwards: refused, with grad mode off too; others pass."""
    import torch
    from tsplat._lib import no_gradients

    plain = torch.zeros(3)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(plain.clone(), torch.ones(3))
        with pytest.raises(ValueError, match="backward or forward"):
            no_gradients(torch, plain, None, dual)
        with torch.no_grad(), pytest.raises(ValueError, match="backward or forward"):
            no_gradients(torch, dual)
        no_gradients(torch, plain, None)
    no_gradients(torch, plain)
    leaf = torch.zeros(3, requires_grad=True)
    with pytest.raises(ValueError, match="backward"):
        no_gradients(torch, leaf)
    with torch.no_grad():
        no_gradients(torch, leaf)


def test_a_load_that_fails_leaves_no_half_of_an_adapter(monkeypatch):
    """An adapter's Linears are loaded one by one: where one fails, for memory or its type, the slot is empty."""
    from types import SimpleNamespace

    import torch
    from tsplat import flow_requests

    lin = {n: SimpleNamespace(in_features=8, out_features=6) for n in ("out", "fc1")}
    model = SimpleNamespace(device="cpu", blocks=[SimpleNamespace(lin=lin)] * 2)
    adapters = flow_requests.FlowAdapters(model, 2, 4)
    good = (torch.ones(3, 8), torch.ones(6, 3))
    weights = {(0, "out"): good, (1, "out"): good, (1, "fc1"): good}
    adapters.load(0, weights)
    adapters.load(1, weights)
    bank = adapters.banks[1]["fc1"]

    def fails(*_):
        raise torch.OutOfMemoryError("no memory")

    monkeypatch.setattr(bank, "load", fails)
    with pytest.raises(torch.OutOfMemoryError):
        adapters.load(1, weights)
    for banks in adapters.banks:
        for b in banks.values():
            assert b.rank.tolist() == [3, 0]
    monkeypatch.undo()
    with pytest.raises(Exception):
        adapters.load(1, {(0, "out"): good, (1, "out"): (good[0], torch.ones(6, 3).to_sparse())})
    for banks in adapters.banks:
        for b in banks.values():
            assert b.rank.tolist() == [3, 0]
