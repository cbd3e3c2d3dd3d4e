"""The flow model over a batch of requests with adapters and latent positions of their own.

The graph is FlowModel.velocity's (flow.py), with two additions: each batch
entry may name a slot of low-rank adapters beside the blocks' packed Linears
(FlowAdapters), and the latent tokens' rotary positions may have several axes
(time, height, width) and differ from request to request (qkv.RopeAxes).
An adapter's part has to be added before what follows the projection, so the
GEMM's fused epilogues do not apply: a Linear stores its projection,
low_rank_add adds to it in place, and the step after it is a pass of its own
-- qkv_rope_axes for the self attention's q/k/v, residual_norm for each
branch's gated residual together with the next branch's norm.
"""
from __future__ import annotations

from . import block_ops as bo
from .adapters import AdapterBank, low_rank_add
from .native_sdpa_ctypes import native_sdpa_f32_ex
from .qkv import qkv_rope_axes


class FlowAdapters:
    """Slots of adapters for the blocks' Linears of a FlowModel: one AdapterBank for each Linear that any adapter
    has loaded (the others cost nothing)."""

    def __init__(self, model, slots, max_rank, dtype=None):
        self.slots, self.max_rank, self.dtype = int(slots), int(max_rank), dtype
        self.device = model.device
        self._sizes = [{name: (lin.in_features, lin.out_features) for name, lin in blk.lin.items()}
                       for blk in model.blocks]
        self.banks = [{} for _ in model.blocks]

    def load(self, slot, weights, scale=1.0):
        """Puts one adapter into a slot: weights {(block, Linear name): (down [rank, in], up [out, rank])}, any
        subset of the blocks' Linears (flow.BLOCK_LINEARS); what the slot held before is unloaded."""
        for (block, name), (down, up) in weights.items():  # (all of them before any slot changes)
            if not 0 <= block < len(self.banks) or name not in self._sizes[block]:
                raise ValueError(f"no Linear {name!r} in block {block}")
            in_f, out_f = self._sizes[block][name]
            rank = int(down.shape[0]) if down.dim() == 2 else 0
            if not 1 <= rank <= self.max_rank or tuple(down.shape) != (rank, in_f) or tuple(up.shape) != (out_f, rank):
                raise ValueError(f"the adapter of {name!r} in block {block} must be down [rank, {in_f}], "
                                 f"up [{out_f}, rank] of rank 1..{self.max_rank}")
        self.unload(slot)
        try:
            for (block, name), (down, up) in weights.items():
                bank = self.banks[block].get(name)
                if bank is None:
                    bank = AdapterBank(self.slots, *self._sizes[block][name], self.max_rank, dtype=self.dtype,
                                       device=self.device)
                bank.load(slot, down, up, scale)
                self.banks[block][name] = bank
        except BaseException:
            self.unload(slot)  # (an adapter of some of its Linears is none)
            raise

    def unload(self, slot):
        if not 0 <= int(slot) < self.slots:
            raise ValueError(f"slot {slot} is outside 0..{self.slots - 1}")
        for banks in self.banks:
            for bank in banks.values():
                bank.unload(slot)


def _adapted(lin, x2, bank, rows):
    out = lin(x2)
    return out if bank is None or rows is None else low_rank_add(out, x2, bank, rows, out=out)


def velocity(model, z, cond, t, *, adapters=None, slots=None, positions=None, rope=None, observe=None):
    """z [B, L, C], cond [B, Lc, C], t [B] (already x1000) -> v [B, L, C], as FlowModel.velocity.
    adapters: FlowAdapters, slots: one slot for each batch entry (-1 for none).  positions [L, axes] or
    [B, L, axes] with rope, a RopeAxes of the model's head size: the latent tokens' places; without them the
    token's index on one axis, as in FlowModel.velocity.  Nothing is copied from the host: after one call on the
    stream it can be captured into a HIP graph, which keeps the slots' numbers and reads what they hold when it is
    replayed."""
    torch, cfg = model.torch, model.cfg
    B, L, C = (int(s) for s in z.shape)
    Lc, H = int(cond.shape[1]), cfg.heads
    if (positions is None) != (rope is None):
        raise ValueError("positions and rope go together")
    if (adapters is None) != (slots is None):
        raise ValueError("adapters and slots go together")
    rows = cond_rows = None
    if adapters is not None:
        if len(adapters.banks) != len(model.blocks):
            raise ValueError("these adapters belong to a model of another depth")
        slots = [int(s) for s in slots]
        if len(slots) != B or any(s >= adapters.slots for s in slots):
            raise ValueError(f"slots must be {B} numbers below {adapters.slots}, negative for none")
        # (filled entry by entry: a copy from the host would wait for the stream, and a graph cannot hold it)
        of_entry = torch.empty(B, 1, dtype=torch.int32, device=model.device)
        for b, s in enumerate(slots):
            of_entry[b].fill_(max(s, -1))
        rows, cond_rows = (of_entry.expand(B, n).contiguous().view(-1) for n in (L, Lc))
    if rope is None:
        rope = model.token_rope()
        positions = torch.arange(L, dtype=torch.int32, device=model.device)[:, None]
    t_emb, t_mod = model.timestep(t)
    x = model.input_layer(z.reshape(B * L, C)).view(B, L, C)
    cond2 = cond.reshape(B * Lc, C)
    branch = gate = None  # the last branch's output, not yet added to x, and its gate
    for i, blk in enumerate(model.blocks):
        banks = adapters.banks[i] if adapters is not None else {}

        def linear(name, x2, at=rows):
            return _adapted(blk.lin[name], x2, banks.get(name), at)

        mod = t_mod.clone()  # [B, 6C] = t_mod + shift_table, chunks (shift, scale, gate) x 2
        for b in range(B):
            bo.add_inplace(mod[b], blk.shift_table)
        shift_msa, scale_msa, gate_msa, shift_mlp, scale_mlp, gate_mlp = mod.chunk(6, dim=1)

        # self attention, after the previous block's MLP has joined x
        if branch is None:
            if observe is not None:
                observe(i, x)
            h = bo.layer_norm(x, cfg.ln_eps, scale=scale_msa, shift=shift_msa)
        else:
            _, h = bo.residual_norm(x, branch, gate=gate, eps=cfg.ln_eps, scale=scale_msa, shift=shift_msa, out=x,
                                    normed=branch)
            if observe is not None:
                observe(i, x)
        qkv = linear("qkv", h.view(B * L, C))
        q, k, v = qkv_rope_axes(qkv, positions, rope, blk.q_gamma, blk.k_gamma, B, L, H)
        a = native_sdpa_f32_ex(q, k, v, out_layout="blhd", precision=model.attention_precision)
        branch = linear("out", a.view(B * L, C)).view(B, L, C)

        # cross attention to the condition tokens (no RoPE)
        _, h = bo.residual_norm(x, branch, gate=gate_msa, weight=blk.xnorm_w, bias=blk.xnorm_b, eps=cfg.ln_eps,
                                out=x, normed=branch)
        xq = bo.head_rmsnorm(linear("xq", h.view(B * L, C)), blk.xq_gamma, B, L, H)
        kv = linear("xkv", cond2, cond_rows)  # [B*Lc, 2C] = [k | v]
        xk = bo.head_rmsnorm(kv, blk.xk_gamma, B, Lc, H, token_stride=2 * C)
        xv = bo.head_rmsnorm(kv[:, C:], None, B, Lc, H, token_stride=2 * C, normalize=False)
        a = native_sdpa_f32_ex(xq, xk, xv, out_layout="blhd", precision=model.attention_precision)
        branch = linear("xout", a.view(B * L, C)).view(B, L, C)

        # MLP
        _, h = bo.residual_norm(x, branch, eps=cfg.ln_eps, scale=scale_mlp, shift=shift_mlp, out=x, normed=branch)
        f = linear("fc1", h.view(B * L, C))
        branch, gate = linear("fc2", bo.gelu_tanh(f, out=f)).view(B, L, C), gate_mlp

    fs = t_emb[:, None, :].expand(B, 2, C).contiguous()  # [B, (shift, scale), C]
    for b in range(B):
        bo.add_inplace(fs[b], model.final_shift_table)
    if branch is None:
        h = bo.layer_norm(x, cfg.final_ln_eps, scale=fs[:, 1], shift=fs[:, 0])
    else:
        _, h = bo.residual_norm(x, branch, gate=gate, eps=cfg.final_ln_eps, scale=fs[:, 1], shift=fs[:, 0], out=x,
                                normed=branch)
    if observe is not None:
        observe(len(model.blocks), x)
    return model.out_layer(h.view(B * L, C)).view(B, L, C)
