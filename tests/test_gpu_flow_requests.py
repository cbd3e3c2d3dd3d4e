"""The flow model over requests with adapters and positions of their own:
its operators together, against a plain 64-bit form of the whole graph."""
from __future__ import annotations

import math

import pytest

from _request_cases import residual_norm, rope as plain_rope

pytestmark = pytest.mark.gpu

SECTIONS = [10, 11, 11]


def _model(cuda, blocks=2, hidden=128, L=90, Lc=33):
    from tsplat.flow import FlowConfig, FlowModel

    cfg = FlowConfig(hidden=hidden, heads=hidden // 64, blocks=blocks, latent_tokens=L, cond_tokens=Lc)
    return FlowModel(cfg, cuda)


def _inputs(torch, cuda, cfg, B, seed):
    g = torch.Generator(device=cuda).manual_seed(seed)
    z = torch.randn(B, cfg.latent_tokens, cfg.hidden, generator=g, device=cuda)
    c = torch.randn(B, cfg.cond_tokens, cfg.hidden, generator=g, device=cuda)
    t = torch.rand(B, generator=g, device=cuda) * 1000
    pos = torch.randint(0, 60, (B, cfg.latent_tokens, 3), generator=g, device=cuda, dtype=torch.int32)
    return z, c, t, pos, g


def _adapter(torch, cuda, model, g, rank, names):
    return {(i, n): (torch.randn(rank, blk.lin[n].in_features, generator=g, device=cuda) / blk.lin[n].in_features ** 0.5,
                     torch.randn(blk.lin[n].out_features, rank, generator=g, device=cuda) * 0.1)
            for i, blk in enumerate(model.blocks) for n in names}


def _plain(torch, model, z, cond, t, loaded, slots, positions, sections):
    """The graph in 64 bits from the decoded packed weights; loaded: {slot: (weights, scale)}."""
    from tsplat.flow import timestep_embedding
    from tsplat.nf24 import decode_nf24_i16_weight_t

    cfg = model.cfg
    B, L, C = z.shape
    H, D = cfg.heads, cfg.head_dim

    def linear(lin, x, at=None):
        w = decode_nf24_i16_weight_t(lin.code01_t, lin.q2_t, lin.scale).double()
        out = x.reshape(-1, x.shape[-1]) @ w + lin.bias.double()
        out = out.reshape(*x.shape[:-1], -1)
        if at is not None:
            for b, slot in enumerate(slots):
                if slot in loaded and at in loaded[slot][0]:
                    (down, up), scale = loaded[slot][0][at], loaded[slot][1]
                    out[b] += scale * ((x[b] @ down.double().t().contiguous()) @ up.double().t().contiguous())
        return out

    def norm(x, eps, scale=None, shift=None, w=None, b=None):
        return residual_norm(torch, x, torch.zeros_like(x), None, 1.0, None, None, None, 0.0, "layer", w, b, eps, scale,
                             shift)[1]

    def head_norm(x, gamma):  # [B, L, H, D]
        return x * math.sqrt(D) / x.norm(dim=-1, keepdim=True).clamp_min(1e-12) * gamma.double()

    def attention(q, k, v):  # [B, H, L, D]
        s = torch.softmax((q @ k.transpose(2, 3).contiguous()) / 8.0, dim=-1)
        return (s @ v).transpose(1, 2).reshape(q.shape[0], q.shape[2], H * D)

    silu = lambda v: v / (1 + torch.exp(-v))  # noqa: E731
    gelu = lambda v: 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))  # noqa: E731
    emb = timestep_embedding(torch, t, cfg.freq_dim, model.device).double()
    t_emb = linear(model.t_fc2, silu(linear(model.t_fc1, emb)))
    t_mod = linear(model.adaln, silu(t_emb))
    x = linear(model.input_layer, z.double())
    cond = cond.double()
    for i, blk in enumerate(model.blocks):
        sh1, sc1, g1, sh2, sc2, g2 = (t_mod + blk.shift_table.double()).chunk(6, 1)
        qkv = linear(blk.lin["qkv"], norm(x, cfg.ln_eps, sc1, sh1), (i, "qkv")).view(B, L, 3, H, D)
        q, k = (plain_rope(torch, qkv[:, :, j], positions, sections, cfg.rope_theta, False, True, gm, 1e-12)[0]
                for j, gm in ((0, blk.q_gamma), (1, blk.k_gamma)))
        a = attention(q, k, qkv[:, :, 2].transpose(1, 2))
        x = x + g1[:, None] * linear(blk.lin["out"], a, (i, "out"))
        h = norm(x, cfg.ln_eps, None, None, blk.xnorm_w, blk.xnorm_b)
        q = head_norm(linear(blk.lin["xq"], h, (i, "xq")).view(B, L, H, D), blk.xq_gamma)
        kv = linear(blk.lin["xkv"], cond, (i, "xkv")).view(B, -1, 2, H, D)
        k = head_norm(kv[:, :, 0], blk.xk_gamma)
        a = attention(*(v.transpose(1, 2) for v in (q, k, kv[:, :, 1])))
        x = x + linear(blk.lin["xout"], a, (i, "xout"))
        f = gelu(linear(blk.lin["fc1"], norm(x, cfg.ln_eps, sc2, sh2), (i, "fc1")))
        x = x + g2[:, None] * linear(blk.lin["fc2"], f, (i, "fc2"))
    shift, scale = (model.final_shift_table.double() + t_emb[:, None]).unbind(1)
    return linear(model.out_layer, norm(x, cfg.final_ln_eps, scale, shift))


def _rel(got, want):
    return float((got.double() - want).norm() / want.norm())


# The packed model's own velocity is held to 2e-6 a block against a plain form (test_gpu_flow); these graphs are two
# blocks, with a projection's worth more of fp32 steps for each adapter.
LIMIT = 1e-5


def test_requests_of_three_kinds(cuda, hiplib):
    """One entry with a fine-tune of every Linear, one without, one of two Linears; positions of three axes."""
    import torch
    from tsplat.flow_requests import FlowAdapters
    from tsplat.qkv import RopeAxes

    model = _model(cuda)
    z, c, t, pos, g = _inputs(torch, cuda, model.cfg, 3, 1)
    every = ["qkv", "out", "xq", "xkv", "xout", "fc1", "fc2"]
    loaded = {2: (_adapter(torch, cuda, model, g, 12, every), 0.5), 0: (_adapter(torch, cuda, model, g, 5, ["qkv", "fc2"]), 2.0)}
    adapters = FlowAdapters(model, 4, 16)
    for slot, (weights, scale) in loaded.items():
        adapters.load(slot, weights, scale)
    rope = RopeAxes(64, SECTIONS, device=cuda)
    slots = [2, -1, 0]
    got = model.velocity(z, c, t, adapters=adapters, slots=slots, positions=pos, rope=rope)
    want = _plain(torch, model, z, c, t, loaded, slots, pos, SECTIONS)
    bare = _plain(torch, model, z, c, t, {}, slots, pos, SECTIONS)
    rel = [_rel(got[b], want[b]) for b in range(3)]
    print({"rel": rel, "without": _rel(got[0], bare[0])})
    assert max(rel) <= LIMIT
    assert _rel(got[0], bare[0]) > 1e-2 and _rel(got[2], bare[2]) > 1e-3
    # another order of the same requests, and each by itself
    swap = [2, 0, 1]
    again = model.velocity(z[swap], c[swap], t[swap], adapters=adapters, slots=[slots[i] for i in swap],
                           positions=pos[swap], rope=rope)
    assert _rel(again, got[swap].double()) <= LIMIT
    adapters.unload(2)
    got = model.velocity(z, c, t, adapters=adapters, slots=slots, positions=pos, rope=rope)
    assert _rel(got[0], bare[0]) <= LIMIT and _rel(got[2], want[2]) <= LIMIT


def test_without_anything_it_is_the_models_velocity(cuda, hiplib):
    """Token indices on one axis and no adapter: FlowModel.velocity's result, by another route."""
    import torch
    from tsplat import flow_requests
    from tsplat.flow_requests import FlowAdapters

    model = _model(cuda, blocks=3)
    z, c, t, _, _ = _inputs(torch, cuda, model.cfg, 2, 2)
    want = model.velocity(z, c, t)
    seen = []
    got = flow_requests.velocity(model, z, c, t, observe=lambda i, x: seen.append((i, x.clone())))
    assert _rel(got, want.double()) <= 1.5 * LIMIT
    states = []
    model.velocity(z, c, t, observe=lambda i, x: states.append((i, x.clone())))
    assert [i for i, _ in seen] == [i for i, _ in states] == [0, 1, 2, 3]
    for (_, a), (_, b) in zip(seen, states):
        assert _rel(a, b.double()) <= 1.5 * LIMIT
    assert torch.equal(model.velocity(z, c, t, adapters=FlowAdapters(model, 2, 8), slots=[1, -1]), got)


def test_a_sampler_step_of_a_request(cuda, hiplib):
    """euler_cfg_step passes a request's adapter and positions on: the guided pair's velocities, joined as ever."""
    import torch
    from tsplat.flow_requests import FlowAdapters
    from tsplat.qkv import RopeAxes

    model = _model(cuda)
    z, c, _, pos, g = _inputs(torch, cuda, model.cfg, 1, 6)
    adapters = FlowAdapters(model, 1, 8, torch.bfloat16)
    adapters.load(0, _adapter(torch, cuda, model, g, 8, ["qkv", "out", "fc1"]))
    request = dict(adapters=adapters, slots=[0, 0], positions=pos[0], rope=RopeAxes(64, SECTIONS, device=cuda))
    z_next, v = model.euler_cfg_step(z[0], c[0], **request)
    ts = model.schedule()
    t = torch.full((2,), ts[0] * 1000.0, device=cuda)
    pair = model.velocity(z.expand(2, -1, -1).contiguous(), torch.cat((c, torch.zeros_like(c))), t, **request)
    want = 3.0 * pair[0].double() - 2.0 * pair[1].double()
    assert _rel(v, want) <= 1e-6
    assert _rel(z_next, z[0].double() - (ts[0] - ts[1]) * v.double()) <= 1e-6
    assert _rel(v, model.euler_cfg_step(z[0], c[0])[1].double()) > 1e-3


def test_a_captured_block_of_requests(cuda, hiplib):
    """The three operators and the projections between them, captured and replayed with eager work between."""
    import torch
    from tsplat import block_ops as bo
    from tsplat.adapters import AdapterBank, adapter_rows, low_rank_add
    from tsplat.qkv import RopeAxes, qkv_rope_axes

    model = _model(cuda, blocks=1)
    cfg, blk = model.cfg, model.blocks[0]
    B, L, C, H = 2, cfg.latent_tokens, cfg.hidden, cfg.heads
    z, _, _, pos, g = _inputs(torch, cuda, cfg, B, 3)
    bank = AdapterBank(2, C, 3 * C, 8, torch.bfloat16, cuda)
    bank.load(1, torch.randn(8, C, generator=g, device=cuda) / 16, torch.randn(3 * C, 8, generator=g, device=cuda))
    rows = adapter_rows([L, L], [1, -1], cuda)
    rope = RopeAxes(64, SECTIONS, device=cuda)
    lin = blk.lin["qkv"]
    qkv = torch.empty(B * L, 3 * C, device=cuda)
    outs = [torch.empty(B, H, L, 64, device=cuda) for _ in range(3)]
    x, y = torch.empty_like(z), torch.empty_like(z)

    def step():
        lin(z.view(B * L, C), out=qkv)
        low_rank_add(qkv, z.view(B * L, C), bank, rows, out=qkv)
        qkv_rope_axes(qkv, pos, rope, blk.q_gamma, blk.k_gamma, B, L, H, outs=outs)
        bo.residual_norm(z, outs[2].view(B, L, C), out=x, normed=y, norm="rms")

    step()
    want = [v.clone() for v in (qkv, *outs, x, y)]
    side = torch.cuda.Stream(device=cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize(cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for _ in range(5):
        for v in (qkv, *outs, x, y):
            v.fill_(float("nan"))
        torch.cuda.synchronize(cuda)
        graph.replay()
        torch.cuda.synchronize(cuda)
        for v, w in zip((qkv, *outs, x, y), want):
            assert torch.equal(v, w)
        low_rank_add(qkv, z.view(B * L, C), bank, rows)


@pytest.mark.parametrize("places", [False, True])
def test_the_model_over_requests_waits_for_nothing(cuda, hiplib, places):
    """velocity() copies nothing from the host, so a call neither waits for the stream nor stays out of a graph: captured,
    with the slots as they were then, and replayed with eager calls of other slots between."""
    import torch
    from tsplat.flow_requests import FlowAdapters
    from tsplat.qkv import RopeAxes

    model = _model(cuda)
    z, c, t, pos, g = _inputs(torch, cuda, model.cfg, 3, 7)
    adapters = FlowAdapters(model, 3, 8)
    for slot in (0, 2):
        adapters.load(slot, _adapter(torch, cuda, model, g, 8, ["qkv", "xkv", "fc2"]))
    kw = dict(adapters=adapters, slots=[2, -1, 0])
    if places:
        kw |= dict(positions=pos, rope=RopeAxes(64, SECTIONS, device=cuda))
    want = model.velocity(z, c, t, **kw)
    other = model.velocity(z, c, t, **(kw | dict(slots=[0, 2, -5])))
    assert _rel(want, other.double()) > 1e-3
    alone = model.velocity(z[:1], c[:1], t[:1], **(kw | dict(slots=[2]) | (dict(positions=pos[0]) if places else {})))
    assert _rel(alone, want[:1].double()) <= LIMIT
    torch.cuda.set_sync_debug_mode("error")
    try:
        again = model.velocity(z, c, t, **kw)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert torch.equal(again, want)
    side = torch.cuda.Stream(device=cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        model.velocity(z, c, t, **kw)  # (the stream's workspaces)
    torch.cuda.synchronize(cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = model.velocity(z, c, t, **kw)
    for _ in range(4):
        got.fill_(float("nan"))
        torch.cuda.synchronize(cuda)
        graph.replay()
        torch.cuda.synchronize(cuda)
        assert torch.equal(got, want)
        assert torch.equal(model.velocity(z, c, t, **(kw | dict(slots=[0, 2, -5]))), other)


def test_two_threads_on_two_streams(cuda, hiplib):
    """The operators keep nothing between calls: two host threads, each on a stream of its own, get what one gets."""
    import threading

    import torch
    from tsplat import block_ops as bo
    from tsplat.adapters import AdapterBank, low_rank_add
    from tsplat.qkv import RopeAxes, rope_axes

    def inputs(seed):
        g = torch.Generator(device=cuda).manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
        bank = AdapterBank.stack(r(3, 40, 256).half(), r(3, 256, 40).half(), [1.0, 0.5, 2.0])
        rows = torch.randint(-1, 3, (900,), generator=g, device=cuda, dtype=torch.int32)
        pos = torch.randint(0, 99, (900, 2), generator=g, device=cuda, dtype=torch.int32)
        return r(900, 256), r(900, 256), bank, rows, pos, RopeAxes(64, [16, 16], device=cuda)

    def step(x, y, bank, rows, pos, rope):
        a = low_rank_add(y, x, bank, rows)
        b, c = bo.residual_norm(x, a, norm="rms")
        return a, b, c, rope_axes(c.view(1, 900, 4, 64), pos, rope)

    sets = [inputs(s) for s in (1, 2)]
    wants = [step(*s) for s in sets]
    torch.cuda.synchronize(cuda)
    wrong = []

    def work(i):
        stream = torch.cuda.Stream(device=cuda)
        with torch.cuda.stream(stream):
            for n in range(40):
                got = step(*sets[i])
                stream.synchronize()
                if not all(torch.equal(p, q) for p, q in zip(got, wants[i])):
                    wrong.append((i, n))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


def test_refusals(cuda, hiplib):
    import torch
    from tsplat.flow_requests import FlowAdapters
    from tsplat.qkv import RopeAxes

    model = _model(cuda, blocks=1)
    z, c, t, pos, g = _inputs(torch, cuda, model.cfg, 2, 4)
    adapters = FlowAdapters(model, 2, 4)
    rope = RopeAxes(64, SECTIONS, device=cuda)
    for kw in (dict(adapters=adapters), dict(slots=[0, 0]), dict(positions=pos), dict(rope=rope),
               dict(adapters=adapters, slots=[0]), dict(adapters=adapters, slots=[0, 2]),
               dict(positions=pos[:, :5], rope=rope), dict(positions=pos, rope=RopeAxes(32, [6, 5, 5], device=cuda)),
               dict(adapters=FlowAdapters(_model(cuda, blocks=2), 2, 4), slots=[0, 0])):
        with pytest.raises(ValueError):
            model.velocity(z, c, t, **kw)
    good = (torch.zeros(4, 128, device=cuda), torch.zeros(128, 4, device=cuda))
    for weights in ({(1, "out"): good}, {(0, "proj"): good}, {(0, "fc1"): good}, {(0, "out"): (good[0], good[0])}):
        with pytest.raises(ValueError):
            adapters.load(0, weights)
    with pytest.raises(ValueError):
        adapters.load(2, {})


def test_tangents_are_refused(cuda, hiplib):
    import torch
    from tsplat.adapters import AdapterBank, low_rank_add
    from tsplat.block_ops import residual_norm
    from tsplat.qkv import RopeAxes, qkv_rope_axes, rope_axes

    x, w = torch.randn(4, 192, device=cuda), torch.ones(192, device=cuda)
    bank, rows = AdapterBank(1, 192, 192, 8, device=cuda), torch.zeros(4, dtype=torch.int32, device=cuda)
    rope, pos = RopeAxes(64, [32], device=cuda), torch.arange(4, dtype=torch.int32, device=cuda)[:, None]
    gamma = torch.ones(1, 64, device=cuda)
    with torch.autograd.forward_ad.dual_level():
        def dual(t):
            return torch.autograd.forward_ad.make_dual(t.clone(), torch.ones_like(t))

        for call in (lambda: low_rank_add(dual(x), x, bank, rows), lambda: low_rank_add(x, dual(x), bank, rows),
                     lambda: residual_norm(dual(x), x), lambda: residual_norm(x, dual(x)),
                     lambda: residual_norm(x, x, weight=dual(w)), lambda: residual_norm(x, x, gate=dual(w[None])),
                     lambda: rope_axes(dual(x).view(1, 4, 3, 64), pos, rope),
                     lambda: qkv_rope_axes(x, pos, rope, dual(gamma), gamma, 1, 4, 1),
                     lambda: qkv_rope_axes(dual(x), pos, rope, gamma, gamma, 1, 4, 1)):
            with pytest.raises(ValueError, match="forward"):
                call()
        low_rank_add(x, x, bank, rows)
        residual_norm(x, x)
