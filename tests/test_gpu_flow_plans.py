"""What the flow model refuses of conditions and their plans, and what it does not do for each entry."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


def _model(cuda, blocks=1, L=40):
    from tsplat.flow import FlowConfig, FlowModel

    return FlowModel(FlowConfig(hidden=128, heads=2, blocks=blocks, latent_tokens=L, cond_tokens=33), cuda)


def _inputs(torch, cuda, lengths, seed=1, L=40):
    g = torch.Generator(device=cuda).manual_seed(seed)
    B = len(lengths)
    z = torch.randn(B, L, 128, generator=g, device=cuda)
    return z, torch.randn(sum(lengths), 128, generator=g, device=cuda), torch.rand(B, generator=g, device=cuda) * 1000


def test_plan_of_another_attention_precision(cuda, hiplib):
    """A plan made for one precision of the attention's products does not serve another in silence."""
    import torch

    model = _model(cuda)
    z, c, t = _inputs(torch, cuda, [20, 5])
    plans = {}
    for precision in ("bf16", "bf16x3", "fp32"):
        model.set_precision(precision, include=("attention",))
        plans[precision] = model.condition_plan(40, [20, 5])
    for now in plans:
        model.set_precision(now, include=("attention",))
        for made, plan in plans.items():
            if made == now:
                assert torch.isfinite(model.velocity(z, c, t, cond_plan=plan)).all()
            else:
                with pytest.raises(ValueError, match="precision"):
                    model.velocity(z, c, t, cond_plan=plan)


def test_refused_before_anything_runs(cuda, hiplib, monkeypatch):
    """A condition that does not fit the batch is refused by its shape, before the first kernel."""
    import torch
    from tsplat.flow_requests import FlowAdapters

    model = _model(cuda)
    z, c, t = _inputs(torch, cuda, [20, 20])
    plan, adapters = model.condition_plan(40, [20, 20]), FlowAdapters(model, 2, 4)

    def never(_):
        raise AssertionError("a kernel ran")

    monkeypatch.setattr(model, "timestep", never)
    wide = torch.zeros(2, 20, 64, device=cuda)
    for cond in (c[None, :20], c.view(1, 40, 128), c, c.view(4, 10, 128), wide, c[0]):
        for kwargs in ({}, dict(adapters=adapters, slots=[0, -1])):
            with pytest.raises(ValueError):
                model.velocity(z, cond, t, **kwargs)
    for cond in (c[:39], c.view(2, 20, 128), c[:, :64], c.view(80, 64)):
        with pytest.raises(ValueError):
            model.velocity(z, cond, t, cond_plan=plan)
    with pytest.raises(AssertionError):
        model.velocity(z, c, t, cond_plan=plan)


def test_condition_split_into_heads(cuda, hiplib):
    """[entries, rows, heads, 64] is the same memory as [entries, rows, C], and taken alike by both routes."""
    import torch

    model = _model(cuda)
    z, c, t = _inputs(torch, cuda, [20, 20])
    positions = torch.arange(40, dtype=torch.int32, device=cuda)[:, None]
    for precision in ("fp32", "fp8"):
        model.set_precision(precision)
        for kwargs in ({}, dict(positions=positions, rope=model.token_rope())):
            want = model.velocity(z, c.view(2, 20, 128), t, **kwargs)
            assert torch.equal(model.velocity(z, c.view(2, 20, 2, 64), t, **kwargs), want)


def test_one_fill_for_each_entry(cuda, hiplib):
    """Conditions of one length: the entries' slots are written once and spread to both kinds of rows."""
    import torch
    from torch.utils._python_dispatch import TorchDispatchMode
    from tsplat.flow_requests import FlowAdapters

    class Fills(TorchDispatchMode):
        count = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.count += "fill_" in func.name()
            return func(*args, **(kwargs or {}))

    model = _model(cuda)
    adapters = FlowAdapters(model, 2, 4)
    counts = {}
    for B in (2, 9):
        z, c, t = _inputs(torch, cuda, [20] * B)
        with Fills() as fills:
            model.velocity(z, c.view(B, 20, 128), t, adapters=adapters, slots=[0] * B)
        counts[B] = fills.count
    assert counts[9] - counts[2] == 7, counts


def test_eight_bits_of_the_other_linears(cuda, hiplib):
    """Precision "fp8" of the timestep, input and output Linears, alone and with the blocks, in both models."""
    import torch
    from tsplat.flow import FlowConfig
    from tsplat.flow_joint import JointFlowModel

    model = _model(cuda, blocks=2)
    z, c, t = _inputs(torch, cuda, [33, 33])
    joint = JointFlowModel(FlowConfig(hidden=128, heads=2, blocks=2, latent_tokens=40, cond_tokens=33), cuda)
    cam = torch.randn(1, 5, generator=torch.Generator(device=cuda).manual_seed(3), device=cuda)
    for m, args in ((model, (z, c.view(2, 33, 128), t)), (joint, (z[0], c[:33], cam, t[:1]))):
        before = m.velocity(*args)
        for include in (("io",), ("blocks", "io")):
            m.set_precision("fp8", include=include)
            got = m.velocity(*args)
            m.set_precision("fp32", include=include)
            for a, b in zip(*((x if isinstance(x, tuple) else (x,)) for x in (got, before))):
                # (a few per cent a Linear; other results than fp32's)
                assert 1e-4 < float((a.double() - b.double()).norm() / b.double().norm()) < 0.3
        after = m.velocity(*args)
        for a, b in zip(*((x if isinstance(x, tuple) else (x,)) for x in (after, before))):
            assert torch.equal(a, b)
