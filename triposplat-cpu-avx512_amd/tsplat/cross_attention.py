"""Cross attention of a batch of requests that bring encoder states of their own lengths.

The queries of all requests lie one after the other, and so do their states: nothing is padded.  CrossPlan says once, for
as long as the lengths stay, which workgroup takes which rows and keys; cross_attention runs it (kernels in
csrc/cross_attention_kernel.h).  native_sdpa_ctypes.native_sdpa_f32_ex is the form of one length for the whole batch.
"""
from __future__ import annotations

import ctypes
import math

from ._lib import check_status, enqueue, load_library, made_on, no_gradients, used_here
from .fp8 import type_ids
from .nf24 import precision_id

HEADER_INTS = 16
MAX_SCALE = 2.3e38  # times log2 e within fp32
# where the header holds the plan's items and the sums of its lengths
_ITEMS, _ROWS, _STATES = 2, 5, 6


def _lengths(name, values):
    out = [int(n) for n in values]
    if any(n < 0 or n >= 1 << 31 for n in out):
        raise ValueError(f"{name} must not be negative, and stay below 2^31")
    return out


class CrossPlan:
    """Which rows of a batch attend to which states: request i's q_lengths[i] query rows to its k_lengths[i] states,
    in order; either may be 0.  Query head h reads key head h / (heads / kv_heads).

    dtype: the type of q, k, v and the result, torch.float32 (default), bfloat16 or float16.  precision: of fp32
    products, "fp32" or the opt-in "bf16x3" / "bf16" (tsplat.nf24.PRECISIONS).  Making one copies it to the GPU and
    waits for that, so it is not made while a graph is captured; calls only read it, and any number of them on any
    streams may share it.  A captured graph reads it too: keep the plan as long as the graph."""

    def __init__(self, q_lengths, k_lengths, heads, head_dim, *, kv_heads=None, dtype=None, precision="fp32",
                 device=None, library=None):
        import torch

        self.q_lengths, self.k_lengths = _lengths("q_lengths", q_lengths), _lengths("k_lengths", k_lengths)
        requests = len(self.q_lengths)
        if len(self.k_lengths) != requests:
            raise ValueError(f"{requests} query lengths and {len(self.k_lengths)} key lengths")
        self.heads, self.head_dim = int(heads), int(head_dim)
        self.kv_heads = self.heads if kv_heads is None else int(kv_heads)
        self.dtype = torch.float32 if dtype is None else dtype
        if self.dtype not in type_ids(torch):
            raise ValueError("dtype is torch.float32, bfloat16 or float16")
        if not 1 <= self.kv_heads <= self.heads < 1 << 16 or self.heads % self.kv_heads:
            raise ValueError(f"{self.heads} heads are not a multiple of {self.kv_heads} key heads, or too many")
        if not 1 <= self.head_dim <= 128:
            raise ValueError(f"head_dim is 1..128, not {self.head_dim}")
        self.precision = precision
        terms = precision_id(precision)
        if terms and self.dtype is not torch.float32:
            raise ValueError("precision is of fp32 products")
        self.library = load_library(library)
        self.device = torch.device("cuda" if device is None else device)
        if self.device.type != "cuda":
            raise ValueError("the plan is for a GPU")
        lengths = [(ctypes.c_int32 * max(1, requests))(*n) for n in (self.q_lengths, self.k_lengths)]
        sizes = (*lengths, requests, self.heads, self.kv_heads, self.head_dim, type_ids(torch)[self.dtype], terms)
        index = torch.cuda.current_device() if self.device.index is None else self.device.index
        with torch.cuda.device(index):
            ints = self.library.tsplat_cross_plan(*sizes, None, 0)
            if ints < 0:
                raise ValueError("too many requests, rows or states for one plan")
            plan = torch.empty(ints, dtype=torch.int32)
            check_status(min(0, self.library.tsplat_cross_plan(*sizes, plan.data_ptr(), ints)), "tsplat_cross_plan")
            self._plan, self._stream = plan.to(torch.device("cuda", index)), made_on(index)
        self.device, self.index = self._plan.device, index
        self._header = (ctypes.c_int32 * HEADER_INTS)(*plan[:HEADER_INTS].tolist())
        self.rows, self.states = self._header[_ROWS], self._header[_STATES]
        # what a call would otherwise look up each time
        self._plan_ptr, self._header_ptr = self._plan.data_ptr(), ctypes.addressof(self._header)
        self._scratch_bytes = self.library.tsplat_cross_scratch_bytes(self._header)
        self._scale = 1.0 / math.sqrt(self.head_dim)


def _vectors(torch, name, t, plan, heads, least):
    """(pointer, token stride, head stride) of [tokens, heads, head_dim]."""
    if not (isinstance(t, torch.Tensor) and t.dtype is plan.dtype and t.dim() == 3 and t.get_device() == plan.index):
        raise ValueError(f"{name} must be a [tokens, {heads}, {plan.head_dim}] tensor of {plan.dtype} on the plan's GPU")
    tokens, h, d = t.shape
    if h != heads or d != plan.head_dim or tokens < least:
        raise ValueError(f"{name} must be [{least} or more, {heads}, {plan.head_dim}], its shape is {list(t.shape)}")
    token, head, unit = t.stride()
    if unit != 1 and d > 1:
        raise ValueError(f"{name} must have unit stride within a vector")
    return t.data_ptr(), token, head


def cross_attention(q, k, v, plan, *, key_bias=None, scale=None, out=None):
    """out[t, h] = sum_j softmax_j(scale q[t, h] . k[j, g] + key_bias[j]) v[j, g], g = h / (heads / kv_heads), over the
    states j of the request that row t belongs to; zeros where it has none, or where every bias is -infinity.

    q [rows, heads, head_dim], k, v [states, kv_heads, head_dim]: of the plan's type, unit stride within a vector, the
    other strides free (k and v may be views of one fused projection) as long as no vectors overlap: shared key heads are
    kv_heads, not an expanded tensor; at least as many rows and states as the plan's lengths add up to.  key_bias [states] fp32: a state whose bias is -infinity is not read into any result, whatever it
    holds (one of +infinity or NaN makes its request's results NaN, and one past 2.3e38 of either sign counts as the type's
    largest or lowest).  An infinity in q, or in k or v of a state that counts, may come out as a NaN.  scale:
    head_dim ** -0.5 by default.  out: None for a new tensor like q, its rows behind the last request zero, or a tensor
    that overlaps nothing that is read, whose rows behind the last request stay as they are.
    Sums, maxima and exponents are fp32; fp32 products as the plan's precision says.  With bf16 and fp16 values the weights
    are rounded to that type before they meet v (half a step of each: in bf16 2.2e-3 of the result's norm, with the
    result's own rounding, which alone is 1.7e-3), and q . k is summed before scale is multiplied in.  Runs on torch's current stream;
    capturable into a HIP graph.  No gradients."""
    import torch

    if not isinstance(plan, CrossPlan):
        raise ValueError("plan must be a CrossPlan")
    q_ptr, q_token, q_head = _vectors(torch, "q", q, plan, plan.heads, plan.rows)
    k_ptr, k_token, k_head = _vectors(torch, "k", k, plan, plan.kv_heads, plan.states)
    v_ptr, v_token, v_head = _vectors(torch, "v", v, plan, plan.kv_heads, plan.states)
    no_gradients(torch, q, k, v, key_bias, out)
    bias_ptr = None
    if key_bias is not None:
        if not (isinstance(key_bias, torch.Tensor) and key_bias.dtype is torch.float32 and key_bias.dim() == 1
                and key_bias.shape[0] >= plan.states and key_bias.is_contiguous()
                and key_bias.get_device() == plan.index):
            raise ValueError(f"key_bias must be a contiguous [{plan.states} or more] fp32 tensor on the plan's GPU")
        bias_ptr = key_bias.data_ptr()
    scale = plan._scale if scale is None else float(scale)
    if not 0.0 < scale <= MAX_SCALE:
        raise ValueError(f"scale must be positive and at most {MAX_SCALE}, not {scale}")
    if out is None:
        out = torch.empty((q.shape[0], plan.heads, plan.head_dim), dtype=plan.dtype, device=plan.device)
        if q.shape[0] > plan.rows:
            out[plan.rows:].zero_()
    out_ptr, out_token, out_head = _vectors(torch, "out", out, plan, plan.heads, plan.rows)
    if plan.rows == 0:
        return out
    used_here(torch, plan._plan, plan.index, plan._stream)
    need = plan._scratch_bytes
    scratch = torch.empty(need, dtype=torch.uint8, device=plan.device) if need else None
    enqueue(plan.library, "tsplat_cross_attention_async", plan.index, q_ptr, q_token, q_head, k_ptr, k_token, k_head,
            v_ptr, v_token, v_head, bias_ptr, scale, out_ptr, out_token, out_head, plan._header_ptr, plan._plan_ptr,
            scratch.data_ptr() if need else None, need)
    return out
