"""QKV postprocess and the fused NF24 QKV projection on the device.

Counterparts of scripts/native_qkv_postprocess_v2_avx512.c:45-105
(``triposplat_qkv_rope_rmsnorm_pack_f32_avx512_v2``) and
scripts/gemm_nf24_qkv_direct_avx512.c:87-199
(``triposplat_gemm_nf24_qkv_rope_rmsnorm_pack_f32_avx512``), as called by
scripts/native_qkv_packed_attention_patch_v3.py:93-158: RoPE first, then
RMSNorm (``y * 8 / max(||y||, 1e-12) * gamma``) on q and k; q comes back as
[B, H, L, 64], k and v packed key-contiguous [B, H, 64, L_padded] with the
tail tokens zero -- the layout the packed SDPA consumes.
"""
from __future__ import annotations

import math

from ._lib import check_status, current_stream_handle, enqueue, load_library, no_gradients, rows_of


# bf16 rounding of the stored k and/or v (the K/V sensitivity probe,
# scripts/native_qkv_postprocess_bf16_probe_avx512.c:34-94, whose three builds
# scripts/build_native_qkv_postprocess_bf16_probe_avx512.sh selects with
# BF16_TARGET): None stores them exact (the default), "k", "v" or "kv" round
# them to the nearest bf16 after the exact computation.  Per call: no other
# call's numerics change.
KV_BF16_ROUND_MODES = {None: 0, "k": 1, "v": 2, "kv": 3}


def kv_round_id(mode) -> int:
    if mode not in KV_BF16_ROUND_MODES:
        raise ValueError(f"kv_round must be one of {sorted(KV_BF16_ROUND_MODES, key=str)}")
    return KV_BF16_ROUND_MODES[mode]


def padded_length(L: int) -> int:
    return (int(L) + 15) & ~15


def _outputs(torch, B, L, H, Lp, device):
    q = torch.empty((B, H, L, 64), dtype=torch.float32, device=device)
    pk = torch.empty((B, H, 64, Lp), dtype=torch.float32, device=device)
    pv = torch.empty((B, H, 64, Lp), dtype=torch.float32, device=device)
    return q, pk, pv


def _check(torch, name, t):
    if t.device.type != "cuda" or t.dtype != torch.float32 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous fp32 GPU tensor")


def qkv_rope_rmsnorm_pack(qkv, frequencies, q_gamma, k_gamma, B, L, H, *, L_padded=None, kv_round=None,
                          library=None):
    """qkv [B*L, 3*H*64]; frequencies [fb, L, H, 64] (cos, sin pairs), fb in {1, B};
    kv_round: the bf16 probe mode of the stored k/v (None = exact)."""
    import torch

    rnd = kv_round_id(kv_round)
    for name, t in (("qkv", qkv), ("frequencies", frequencies), ("q_gamma", q_gamma), ("k_gamma", k_gamma)):
        _check(torch, name, t)
    Lp = padded_length(L) if L_padded is None else int(L_padded)
    q, pk, pv = _outputs(torch, B, L, H, Lp, qkv.device)
    lib = load_library(library)
    with torch.cuda.device(qkv.device):
        status = lib.tsplat_qkv_postprocess_async(
            qkv.data_ptr(), frequencies.data_ptr(), q_gamma.data_ptr(), k_gamma.data_ptr(),
            q.data_ptr(), pk.data_ptr(), pv.data_ptr(), int(B), int(L), int(H), 64, Lp,
            int(frequencies.shape[0]), rnd, current_stream_handle(qkv.device),
        )
    check_status(status, "tsplat_qkv_postprocess_async")
    return q, pk, pv


def gemm_nf24_qkv_direct(x2, code01_t, q2_t, scale, bias, frequencies, q_gamma, k_gamma, B, L, H, *,
                         L_padded=None, precision="fp32", kv_layout="packed", kv_round=None, planes=None,
                         library=None):
    """NF24 QKV projection of x2 [B*L, K] (N = 3*H*64) then the postprocess;
    precision (and planes) of the projection as tsplat.nf24.nf24_linear.
    kv_layout "packed" returns k/v [B, H, 64, L_padded] (the reference's
    layout), "bhld" returns k/v [B, H, L, 64] like q (what the unpacked SDPA
    reads).  kv_round: the bf16 probe mode of the stored k/v (None = exact)."""
    import torch

    from .nf24 import planes_pointers, precision_id

    mode = precision_id(precision)
    rnd = kv_round_id(kv_round)
    if kv_layout not in ("packed", "bhld"):
        raise ValueError(f"kv_layout must be 'packed' or 'bhld', not {kv_layout!r}")
    for name, t in (("x", x2), ("frequencies", frequencies), ("q_gamma", q_gamma), ("k_gamma", k_gamma)):
        _check(torch, name, t)
    Lp = padded_length(L) if L_padded is None else int(L_padded)
    if kv_layout == "packed":
        q, pk, pv = _outputs(torch, B, L, H, Lp, x2.device)
    else:
        q, pk, pv = (torch.empty((B, H, L, 64), dtype=torch.float32, device=x2.device) for _ in range(3))
    lib = load_library(library)
    with torch.cuda.device(x2.device):
        args = (x2.data_ptr(), code01_t.data_ptr(), q2_t.data_ptr(), scale.data_ptr(), bias.data_ptr(),
                frequencies.data_ptr(), q_gamma.data_ptr(), k_gamma.data_ptr(), q.data_ptr(), pk.data_ptr(),
                pv.data_ptr(), int(B), int(L), int(x2.shape[1]), int(code01_t.shape[1]), int(H), 64, Lp,
                int(frequencies.shape[0]))
        stream = current_stream_handle(x2.device)
        if mode == 0 and kv_layout == "packed" and rnd == 0:
            name, status = "tsplat_gemm_nf24_qkv_direct_async", lib.tsplat_gemm_nf24_qkv_direct_async(*args, stream)
        elif mode != 0 and planes is not None:
            name = "tsplat_gemm_nf24_qkv_direct_planes_async"
            ptrs = planes_pointers(planes, int(x2.shape[1]), int(code01_t.shape[1]), mode)
            status = lib.tsplat_gemm_nf24_qkv_direct_planes_async(*args, int(kv_layout == "bhld"), mode, rnd,
                                                                    *ptrs, stream)
        else:
            name = "tsplat_gemm_nf24_qkv_direct_ex_async"
            status = lib.tsplat_gemm_nf24_qkv_direct_ex_async(*args, int(kv_layout == "bhld"), mode, rnd,
                                                                stream)
    check_status(status, name)
    return q, pk, pv


def q_kv_selected_rope_rmsnorm_pack(q, kv, frequencies, selected_indices, q_gamma, k_gamma, B, Lq, Lk, H,
                                    *, L_padded=None, kv_round=None, library=None):
    """Selected query rows (scripts/native_qkv_postprocess_v2_avx512.c:107-191):
    q [B, Lq, H*64] from a Q-only projection, kv [B, Lk, 2*H*64] = [k | v];
    query t is rotated with frequency row selected_indices[t] (int64 GPU
    tensor).  Returns q [B, H, Lq, 64] and packed k/v [B, H, 64, L_padded].
    kv_round: the bf16 probe mode of the stored k/v (None = exact)."""
    import torch

    rnd = kv_round_id(kv_round)
    for name, t in (("q", q), ("kv", kv), ("frequencies", frequencies), ("q_gamma", q_gamma),
                    ("k_gamma", k_gamma)):
        _check(torch, name, t)
    if (selected_indices.device.type != "cuda" or selected_indices.dtype != torch.int64
            or not selected_indices.is_contiguous() or selected_indices.numel() != int(Lq)):
        raise ValueError("selected_indices must be a contiguous int64 GPU tensor of length Lq")
    Lp = padded_length(Lk) if L_padded is None else int(L_padded)
    qo = torch.empty((B, H, Lq, 64), dtype=torch.float32, device=q.device)
    pk = torch.empty((B, H, 64, Lp), dtype=torch.float32, device=q.device)
    pv = torch.empty((B, H, 64, Lp), dtype=torch.float32, device=q.device)
    lib = load_library(library)
    with torch.cuda.device(q.device):
        status = lib.tsplat_q_kv_selected_postprocess_async(
            q.data_ptr(), kv.data_ptr(), frequencies.data_ptr(), selected_indices.data_ptr(),
            q_gamma.data_ptr(), k_gamma.data_ptr(), qo.data_ptr(), pk.data_ptr(), pv.data_ptr(),
            int(B), int(Lq), int(Lk), int(H), 64, Lp, int(frequencies.shape[0]), rnd,
            current_stream_handle(q.device),
        )
    check_status(status, "tsplat_q_kv_selected_postprocess_async")
    return qo, pk, pv


class RopeAxes:
    """Which position each pair of a head's vector turns by, and how fast: the plan of rope_axes.

    dim: the head's size, even, at most 512; sections: how many of its dim / 2 pairs each axis (time, height, width)
    takes, in order.  An axis has a ramp of its own, frequency theta^(-j / n) of its j-th pair of n; with shared,
    one ramp theta^(-p / (dim / 2)) over all pairs is dealt out to the axes.  interleaved: a pair is the neighbours
    (2p, 2p + 1), as in rope_complex; else (p, p + dim / 2)."""

    def __init__(self, dim, sections, theta=10000.0, *, shared=False, interleaved=True, device="cuda"):
        import torch

        sections = [int(n) for n in sections]
        dim = int(dim)
        if dim < 2 or dim % 2 or dim > 512 or not 1 <= len(sections) <= 8:
            raise ValueError("dim must be even, 2..512, with 1..8 sections")
        if min(sections) < 0 or sum(sections) != dim // 2:
            raise ValueError(f"the sections of {dim // 2} pairs must add up to them, not {sections}")
        if not float(theta) > 0.0:
            raise ValueError("theta must be positive")
        self.dim, self.sections, self.theta = dim, tuple(sections), float(theta)
        self.shared, self.interleaved = bool(shared), bool(interleaved)
        axis = [i for i, n in enumerate(sections) for _ in range(n)]
        if shared:
            ramp = [self.theta ** (-p / (dim // 2)) for p in range(dim // 2)]
        else:
            ramp = [self.theta ** (-j / n) for n in sections for j in range(n)]
        # revolutions per unit of position, in 64 bits: the kernel keeps the fraction of position * turns
        turns = torch.tensor([f / (2.0 * math.pi) for f in ramp], dtype=torch.float64)
        both = torch.cat((turns.view(torch.uint8), torch.tensor(axis, dtype=torch.int32).view(torch.uint8)))
        both = both.to(device)  # (one copy to the device)
        self.turns, self.axis = both[:4 * dim].view(torch.float64), both[4 * dim:].view(torch.int32)
        self.device, self.index, self.axes = self.turns.device, self.turns.get_device(), len(sections)


def _gamma(torch, g, H, D, device):
    if g is None:
        return None
    if not (isinstance(g, torch.Tensor) and g.dtype is torch.float32 and g.shape == (H, D) and g.is_contiguous()
            and g.get_device() == device):
        raise ValueError(f"gamma must be a contiguous [{H}, {D}] fp32 tensor on the GPU of x")
    return g.data_ptr()


def _rope_call(torch, x, strides, parts, gamma0, gamma1, positions, rope, eps, B, L, H, outs, out_bhld, library):
    D, at = rope.dim, x.get_device()
    shape = (B, H, L, D) if out_bhld else (B, L, H, D)
    if outs is None:
        outs = [x.new_empty(shape) for _ in range(parts)]
    else:
        for o in outs:
            if not (isinstance(o, torch.Tensor) and o.dtype is torch.float32 and o.shape == shape
                    and o.is_contiguous() and o.get_device() == at):
                raise ValueError(f"out must be a contiguous {list(shape)} fp32 tensor on the GPU of x")
    if not isinstance(positions, torch.Tensor) or positions.get_device() != at or rope.index != at:
        raise ValueError("x, positions and rope must be on one GPU")
    kind, places = positions.dtype, positions.shape
    fractional, batches = kind is torch.float32, places[0] if len(places) == 3 else 1
    if (not (fractional or kind is torch.int32) or not positions.is_contiguous() or not 2 <= len(places) <= 3
            or places[-2] != L or places[-1] != rope.axes or batches not in (1, B)):
        raise ValueError(f"positions must be a contiguous [{L}, {rope.axes}] or [{B}, {L}, {rope.axes}] tensor of int32 "
                         "or fp32")
    no_gradients(torch, x, positions, gamma0, gamma1, *outs)
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    if H > 1 << 16 or B * L >= 1 << 31:
        raise ValueError("at most 2^16 heads, and fewer than 2^31 tokens")
    gammas = _gamma(torch, gamma0, H, D, at), _gamma(torch, gamma1, H, D, at)
    if B * L * H == 0:
        return outs
    dst = [outs[0].data_ptr(), outs[1].data_ptr(), outs[2].data_ptr()] if parts == 3 else [outs[0].data_ptr(), None, None]
    enqueue(load_library(library), "tsplat_rope_axes_async", at, x.data_ptr(), *strides, parts, *gammas, *dst,
            positions.data_ptr(), fractional, batches, rope.axes, rope.turns.data_ptr(), rope.axis.data_ptr(),
            rope.interleaved, eps, B, L, H, D, out_bhld)
    return outs


def rope_axes(x, positions, rope, *, gamma=None, eps=1.0e-12, out=None, out_bhld=True, library=None):
    """x [B, L, H, D] turned by positions of several axes, then with a gamma [H, D] the per-head RMSNorm
    y * sqrt(D) / max(||y||, eps) * gamma, as [B, H, L, D] (out_bhld) or [B, L, H, D].

    x: fp32 on the GPU, any strides that do not overlap, unit in D (a view into a projection's rows).  positions:
    [L, axes] or [B, L, axes], int32 or fp32 (fractional places); an angle is taken in 64 bits, so far positions
    keep their precision.  rope: RopeAxes.  out may not lie in the memory that x spans, nor over anything else that is
    read.  No gradients."""
    import torch

    if not (isinstance(x, torch.Tensor) and x.is_cuda and x.dtype == torch.float32 and x.dim() == 4):
        raise ValueError("x must be a [B, L, H, D] fp32 GPU tensor")
    B, L, H, D = x.shape
    if not isinstance(rope, RopeAxes) or D != rope.dim:
        raise ValueError(f"rope must be a RopeAxes of the heads' size {D}")
    sb, sl, sh, sd = x.stride()
    if sd != 1:
        raise ValueError("x must have unit stride within its vectors")
    if (B > 1 and sb < D) or (L > 1 and sl < D) or (H > 1 and sh < D):
        raise ValueError("the vectors of x overlap")
    return _rope_call(torch, x, (0, sb, sl, sh), 1, gamma, None, positions, rope, eps, B, L, H,
                      None if out is None else [out], out_bhld, library)[0]


def qkv_rope_axes(qkv, positions, rope, q_gamma, k_gamma, B, L, H, *, eps=1.0e-12, outs=None, library=None):
    """qkv [B*L, 3*H*D] = [q | k | v] of an unfused projection: q and k turned by positions of several axes and
    normed per head as rope_axes does (a gamma of None: turned only), v moved; all three come back as [B, H, L, D],
    what native_sdpa_f32_ex reads.  outs: three such tensors to write, or None.  The rows of qkv may be strided."""
    import torch

    if not isinstance(rope, RopeAxes):
        raise ValueError("rope must be a RopeAxes")
    B, L, H = int(B), int(L), int(H)
    width = H * rope.dim
    rows, stride = rows_of(torch, "qkv", qkv, 3 * width)
    if rows != B * L:
        raise ValueError(f"qkv has {rows} rows, not B * L = {B * L}")
    if outs is not None and len(outs) != 3:
        raise ValueError("outs must be three tensors")
    return tuple(_rope_call(torch, qkv, (width, L * stride, stride, rope.dim), 3, q_gamma, k_gamma, positions,
                            rope, eps, B, L, H, outs, True, library))
