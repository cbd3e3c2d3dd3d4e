"""The flow model over requests whose conditions have lengths of their own, and its Linears in 8 bits: the operators
together, against a plain 64-bit form of the whole graph."""
from __future__ import annotations

import math

import pytest

from _fp8_cases import values
from _request_cases import residual_norm, rope as plain_rope

pytestmark = pytest.mark.gpu

# two blocks of fp32 steps, as the requests' graph is held to (test_gpu_flow_requests)
LIMIT = 1e-5
# An activation that lies within the graph's own error of a border between two codes may fall to either side: about
# 1e-6 / 2^-4 of them, and each moves its Linear's result by 2^-4 / sqrt(values) of its norm; a block of 7 Linears on
# some 10^4 values: sqrt(7e4 * 1.6e-5) * 2^-4 / 1e2 < 1e-3, for two blocks twice that, an order below what 8 bits cost.
LIMIT8 = 4e-3


def _model(cuda, blocks=2, hidden=128, L=90, Lc=33):
    from tsplat.flow import FlowConfig, FlowModel

    return FlowModel(FlowConfig(hidden=hidden, heads=hidden // 64, blocks=blocks, latent_tokens=L, cond_tokens=Lc), cuda)


def _inputs(torch, cuda, model, lengths, seed):
    g = torch.Generator(device=cuda).manual_seed(seed)
    B, cfg = len(lengths), model.cfg
    z = torch.randn(B, cfg.latent_tokens, cfg.hidden, generator=g, device=cuda)
    c = torch.randn(sum(lengths), cfg.hidden, generator=g, device=cuda)
    return z, c, torch.rand(B, generator=g, device=cuda) * 1000, g


def _plain(torch, model, z, cond, lengths, t, loaded=None, slots=None, eight=False):
    """The graph in 64 bits from the decoded packed weights; loaded: {slot: (weights, scale)}; eight: the blocks' weights
    and their Linears' rows in 8 bits."""
    from tsplat.flow import timestep_embedding
    from tsplat.nf24 import decode_nf24_i16_weight, decode_nf24_i16_weight_t

    cfg = model.cfg
    (B, L, C), H, D = z.shape, cfg.heads, cfg.head_dim

    def linear(lin, x, at=None, entry=None):
        w = decode_nf24_i16_weight_t(lin.code01_t, lin.q2_t, lin.scale).double()
        rows = x.reshape(-1, x.shape[-1])
        made = rows
        if eight and at is not None:
            w = values(torch, decode_nf24_i16_weight(lin.code01_t, lin.q2_t, lin.scale)).t().contiguous()
            made = values(torch, rows.float())
        out = (made @ w + lin.bias.double()).reshape(*x.shape[:-1], -1)
        for b, slot in enumerate(slots or ()):
            if at is not None and slot in loaded and at in loaded[slot][0] and entry in (None, b):
                (down, up), scale = loaded[slot][0][at], loaded[slot][1]
                part = slice(None) if entry == b else b
                out[part] += scale * ((x[part] @ down.double().t().contiguous()) @ up.double().t().contiguous())
        return out

    def norm(x, eps, scale=None, shift=None, w=None, b=None):
        return residual_norm(torch, x, torch.zeros_like(x), None, 1.0, None, None, None, 0.0, "layer", w, b, eps, scale,
                             shift)[1]

    def head_norm(x, gamma):  # [..., H, D]
        return x * math.sqrt(D) / x.norm(dim=-1, keepdim=True).clamp_min(1e-12) * gamma.double()

    def attention(q, k, v):  # [H, L, D] -> [L, H D]
        s = torch.softmax((q @ k.transpose(1, 2).contiguous()) / 8.0, dim=-1)
        return (s @ v.contiguous()).transpose(0, 1).reshape(q.shape[1], H * D)

    silu = lambda v: v / (1 + torch.exp(-v))  # noqa: E731
    gelu = lambda v: 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))  # noqa: E731
    t_emb = linear(model.t_fc2, silu(linear(model.t_fc1, timestep_embedding(torch, t, cfg.freq_dim, model.device).double())))
    t_mod = linear(model.adaln, silu(t_emb))
    x = linear(model.input_layer, z.double())
    positions = torch.arange(L, device=model.device)[:, None]
    for i, blk in enumerate(model.blocks):
        sh1, sc1, g1, sh2, sc2, g2 = (t_mod + blk.shift_table.double()).chunk(6, 1)
        qkv = linear(blk.lin["qkv"], norm(x, cfg.ln_eps, sc1, sh1), (i, "qkv")).view(B, L, 3, H, D)
        q, k = (plain_rope(torch, qkv[:, :, j], positions, [D // 2], cfg.rope_theta, False, True, gm, 1e-12)[0]
                for j, gm in ((0, blk.q_gamma), (1, blk.k_gamma)))
        a = torch.stack([attention(q[b], k[b], qkv[b, :, 2].transpose(0, 1)) for b in range(B)])
        x = x + g1[:, None] * linear(blk.lin["out"], a, (i, "out"))
        h = norm(x, cfg.ln_eps, None, None, blk.xnorm_w, blk.xnorm_b)
        q = head_norm(linear(blk.lin["xq"], h, (i, "xq")).view(B, L, H, D), blk.xq_gamma)
        parts, start = [], 0
        for b, n in enumerate(lengths):
            a = torch.zeros(L, C, dtype=torch.float64, device=z.device)
            if n:
                kv = linear(blk.lin["xkv"], cond[start:start + n].double(), (i, "xkv"), b).view(n, 2, H, D)
                a = attention(q[b].transpose(0, 1).contiguous(), head_norm(kv[:, 0], blk.xk_gamma).transpose(0, 1),
                              kv[:, 1].transpose(0, 1))
            parts.append(a)
            start += n
        x = x + linear(blk.lin["xout"], torch.stack(parts), (i, "xout"))
        f = gelu(linear(blk.lin["fc1"], norm(x, cfg.ln_eps, sc2, sh2), (i, "fc1")))
        x = x + g2[:, None] * linear(blk.lin["fc2"], f, (i, "fc2"))
    shift, scale = (model.final_shift_table.double() + t_emb[:, None]).unbind(1)
    return linear(model.out_layer, norm(x, cfg.final_ln_eps, scale, shift))


def _rel(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("lengths", [[33, 0, 7], [1, 257], [0, 0], [50], [40, 40, 40, 40]])
def test_conditions_of_their_own_lengths(cuda, hiplib, lengths):
    import torch

    model = _model(cuda)
    z, c, t, _ = _inputs(torch, cuda, model, lengths, 1)
    plan = model.condition_plan(90, lengths)
    got = model.velocity(z, c, t, cond_plan=plan)
    want = _plain(torch, model, z, c, lengths, t)
    rel = [_rel(got[b], want[b]) for b in range(len(lengths))]
    print({"rel": rel})
    assert max(rel) <= LIMIT
    if len(set(lengths)) == 1 and lengths[0]:  # the batch of one length, by the other route
        same = model.velocity(z, c.view(len(lengths), -1, model.cfg.hidden), t)
        assert _rel(got, same.double()) <= LIMIT


def test_with_adapters(cuda, hiplib):
    """An entry with an adapter of the condition's Linear, one without a condition, one without an adapter."""
    import torch
    from tsplat.flow_requests import FlowAdapters

    model = _model(cuda)
    lengths, slots = [20, 0, 61], [1, 1, -1]
    z, c, t, g = _inputs(torch, cuda, model, lengths, 2)
    names = ["xq", "xkv", "xout", "fc1"]
    weights = {(i, n): (torch.randn(6, blk.lin[n].in_features, generator=g, device=cuda) / blk.lin[n].in_features ** 0.5,
                        torch.randn(blk.lin[n].out_features, 6, generator=g, device=cuda) * 0.1)
               for i, blk in enumerate(model.blocks) for n in names}
    adapters = FlowAdapters(model, 2, 8)
    adapters.load(1, weights, 0.5)
    loaded = {1: (weights, 0.5)}
    plan = model.condition_plan(90, lengths)
    for precision, limit in (("fp32", LIMIT), ("fp8", LIMIT8)):
        model.set_precision(precision)
        got = model.velocity(z, c, t, adapters=adapters, slots=slots, cond_plan=plan)
        want = _plain(torch, model, z, c, lengths, t, loaded, slots, precision == "fp8")
        rel = [_rel(got[b], want[b]) for b in range(3)]
        print({precision: rel})
        assert max(rel) <= limit
    model.set_precision("fp32")


def test_eight_bits(cuda, hiplib):
    """Both routes of the graph in precision "fp8" against the 64-bit form of the same 8-bit rows; back in fp32 the
    results are what they were."""
    import torch

    model = _model(cuda, hidden=192)
    lengths = [33, 33]
    z, c, t, _ = _inputs(torch, cuda, model, lengths, 3)
    cond = c.view(2, 33, -1)
    before = model.velocity(z, cond, t)
    model.set_precision("fp8")
    want = _plain(torch, model, z, c, lengths, t, eight=True)
    for got in (model.velocity(z, cond, t), model.velocity(z, c, t, cond_plan=model.condition_plan(90, lengths))):
        rel = _rel(got, want)
        print({"rel": rel, "to fp32": _rel(got, before.double())})
        assert rel <= LIMIT8 < _rel(got, before.double()) < 0.2
    model.set_precision("fp32")
    assert torch.equal(model.velocity(z, cond, t), before)


def test_packed_linear_in_eight_bits(cuda, hiplib):
    """Every form that the models call: whole, a run of outputs, the epilogues, the fused QKV; and prepared rows."""
    import torch
    from tsplat import block_ops as bo
    from tsplat.flow import PackedLinear, rope_frequencies
    from tsplat.fp8 import fp8_linear, quantize_blocks
    from tsplat.nf24 import decode_nf24_i16_weight
    from tsplat.qkv import qkv_rope_rmsnorm_pack

    lin = PackedLinear.random(torch, 128, 384, 5, cuda)
    lin.set_precision("fp8")
    assert torch.equal(lin.rows8.codes.float(), quantize_blocks(decode_nf24_i16_weight(lin.code01_t, lin.q2_t, lin.scale)).codes.float())
    g = torch.Generator(device=cuda).manual_seed(1)
    for M in (6, 70):
        x = torch.randn(M, 128, generator=g, device=cuda)
        y = lin(x)
        assert torch.equal(y, fp8_linear(x, lin.rows8, lin.bias)) and torch.equal(y, lin(quantize_blocks(x)))
        for start, count in ((0, 128), (128, 256), (5, 77)):
            assert torch.equal(lin(x, output_start=start, output_count=count), y[:, start:start + count])
        assert torch.equal(lin.epilogue(x, bo.EPILOGUE_GELU), fp8_linear(x, lin.rows8, lin.bias, activation="gelu"))
        r = torch.randn(M, 384, generator=g, device=cuda)
        gate = torch.randn(2, 3 * 384, generator=g, device=cuda)[:, 384:768]
        for kind, kwargs, want in ((bo.EPILOGUE_ADD, {}, y + r),
                                   (bo.EPILOGUE_GATED, dict(gate=gate), r + y * gate.repeat_interleave(M // 2, 0))):
            out = r.clone()
            assert lin.epilogue(x, kind, out=out, **kwargs) is out
            # (a product and a sum of a few units, each rounded once)
            assert float((out.double() - want.double()).abs().max()) <= 2.0 ** -22 * float(want.abs().max())
        gamma = torch.rand(2, 64, generator=g, device=cuda) + 0.5
        freqs = rope_frequencies(torch, M // 2, 2, 1e4, cuda)
        got = lin.qkv_direct(x, freqs, gamma, gamma, 2, M // 2, 2, kv_layout=lin.kv_layout)
        for a, b in zip(got, qkv_rope_rmsnorm_pack(y, freqs, gamma, gamma, 2, M // 2, 2)):
            assert torch.equal(a, b)
        with pytest.raises(ValueError):
            lin.qkv_direct(x, freqs, gamma, gamma, 2, M // 2, 2, kv_layout="bhld")
        with pytest.raises(ValueError):
            lin.epilogue(x, bo.EPILOGUE_GATED, out=r)
        with pytest.raises(ValueError):
            lin(x, output_start=300, output_count=100)
    lin.set_precision("fp32")
    assert lin.rows8 is None and lin.kv_layout == "bhld"


def test_joint_model_in_eight_bits(cuda, hiplib):
    import torch
    from tsplat.flow import FlowConfig
    from tsplat.flow_joint import JointFlowModel

    model = JointFlowModel(FlowConfig(hidden=128, heads=2, blocks=3, latent_tokens=90, cond_tokens=33), cuda)
    g = torch.Generator(device=cuda).manual_seed(4)
    z, c, cam = (torch.randn(*s, generator=g, device=cuda) for s in ((90, 128), (33, 128), (1, 5)))
    t = torch.full((1,), 500.0, device=cuda)
    for kwargs in ({}, dict(selected_final=False), dict(compress=True)):
        before = model.velocity(z, c[:1].expand(33, -1).contiguous(), cam, t, **kwargs)
        model.set_precision("fp8")
        got = model.velocity(z, c[:1].expand(33, -1).contiguous(), cam, t, **kwargs)
        model.set_precision("fp32")
        for a, b in zip(got, before):
            assert 1e-4 < _rel(a, b.double()) < 0.2  # (a few per cent a Linear)


def test_captured(cuda, hiplib):
    """A velocity with a condition plan in a graph, eager calls between its replays."""
    import torch

    model = _model(cuda)
    lengths = [33, 0, 300]
    z, c, t, _ = _inputs(torch, cuda, model, lengths, 5)
    plan = model.condition_plan(90, lengths)
    for precision in ("fp32", "fp8"):
        model.set_precision(precision)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            model.velocity(z, c, t, cond_plan=plan)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y = model.velocity(z, c, t, cond_plan=plan)
        for turn in range(4):
            z.mul_(-0.75), c.mul_(1.125)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, model.velocity(z, c, t, cond_plan=plan)), (precision, turn)


def test_refusals(cuda, hiplib):
    import torch

    model = _model(cuda)
    z, c, t, _ = _inputs(torch, cuda, model, [20, 5], 6)
    plan = model.condition_plan(90, [20, 5])
    for args, p in (((z, c[:24], t), plan), ((z, c.view(1, 25, -1), t), plan), ((z[:, :80], c, t), plan),
                    ((z[:1], c, t[:1]), plan), ((z, c, t), model.condition_plan(90, [20, 4])),
                    ((z, c, t), "plan")):
        with pytest.raises(ValueError):
            model.velocity(*args, cond_plan=p)
    for precision in ("fp32", "fp8"):  # one condition for two entries
        model.set_precision(precision)
        with pytest.raises(ValueError):
            model.velocity(z, c[None, :20], t)
    model.set_precision("fp32")
    for include in (("blocks", "attention"), ("attention",)):
        with pytest.raises(ValueError):
            model.set_precision("fp8", include=include)
    assert model.precision == "fp32" and all(lin.precision == "fp32" for b in model.blocks for lin in b.lin.values())
    with pytest.raises(ValueError):
        model.set_precision("fp4")
