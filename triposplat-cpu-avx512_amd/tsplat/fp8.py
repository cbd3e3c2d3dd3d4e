"""Rows in 8 bits with a scale for each block of 128, and a Linear on them.

The matrix cores multiply e4m3 values at twice the rate of bf16 and take a
power-of-two scale for each operand with the instruction.  quantize_blocks
brings the rows of a weight or an activation to that form, one byte a value;
fp8_linear multiplies two of them, fp32 sums, with the step that follows the
projection in the same kernel (kernels in csrc/fp8_quantize.hip and
csrc/fp8_linear.hip).  A value keeps 4 significant bits: a Linear of random
signs is off by about 4 % of its result's norm, which the caller opts into
(flow.FlowModel.set_precision("fp8")).
"""
from __future__ import annotations

from ._lib import enqueue, load_library, made_on, matrix_rows, no_gradients, used_here

BLOCK = 128
# the library's limits
MAX_ROWS = 1 << 27
MAX_FEATURES = 1 << 20

_TYPE_IDS: dict = {}


def type_ids(torch):
    """The library's numbers of the types that rows may have."""
    if not _TYPE_IDS:
        _TYPE_IDS.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
    return _TYPE_IDS


class Fp8Rows:
    """Rows of K values in 8 bits: values [rows, K] = codes * 2^(exponents - 127), an exponent for each 128 of a row.
    Made by quantize_blocks."""

    def __init__(self, buffer, at, rows, features, stream):
        # uint8: the codes' rows, K rounded up to 128 bytes each, and the exponents', blocks rounded up to 4, at `at`
        self._buffer, self._at, self._stream = buffer, at, stream
        self.rows, self.features = rows, features
        self.blocks = -(-features // BLOCK)
        self.device, self.index = buffer.device, buffer.get_device()
        base = buffer.data_ptr()
        self.codes_ptr, self.exponents_ptr = base + at[0], base + at[1]

    def _rows_of(self, which, width, step):
        return self._buffer.as_strided((self.rows, width), (step, 1), self._at[which])

    @property
    def codes(self):
        """[rows, K] float8_e4m3fn, a view."""
        import torch

        return self._rows_of(0, self.features, self.blocks * BLOCK).view(torch.float8_e4m3fn)

    @property
    def exponents(self):
        """[rows, ceil(K / 128)] uint8, a view: a block's scale is 2^(exponent - 127)."""
        return self._rows_of(1, self.blocks, _fours(self.blocks))

    def narrow(self, start, count):
        """Rows start .. start + count - 1, a view (of a weight: a run of its outputs)."""
        if start < 0 or count < 0 or start + count > self.rows:
            raise ValueError(f"rows {start}..{start + count} of {self.rows}")
        at = self._at[0] + start * self.blocks * BLOCK, self._at[1] + start * _fours(self.blocks)
        return Fp8Rows(self._buffer, at, count, self.features, self._stream)

    def dequantize(self):
        """The values that the codes stand for, fp32 [rows, K] (exact)."""
        import torch

        # (2^(e - 127) by its bits in 64 bits: 2^-127 is subnormal in fp32)
        scale = ((self.exponents.to(torch.int64) + 896) << 52).view(torch.float64)
        padded = self._rows_of(0, self.blocks * BLOCK, self.blocks * BLOCK).view(torch.float8_e4m3fn).float()
        padded = padded.unflatten(1, (self.blocks, BLOCK)).double() * scale[:, :, None]
        return padded.float().flatten(1)[:, :self.features].contiguous()


def _fours(n):
    return (n + 3) // 4 * 4


def quantize_blocks(x, *, library=None):
    """The rows of x [..., K] in 8 bits, as Fp8Rows.

    x: fp32, bf16 or fp16 on the GPU, unit column stride and one row stride.  A block's scale is the smallest power of
    two, 2^-127 at least, that brings its largest finite magnitude to 448 or below; a code is the nearest e4m3 value of
    x / scale, ties to even.  An infinity or NaN becomes a NaN and leaves the scale alone.  Runs on torch's current
    stream; capturable into a HIP graph.  No gradients."""
    import torch

    types = type_ids(torch)
    kind = x.dtype if isinstance(x, torch.Tensor) else None
    if kind not in types:
        raise ValueError("x must be an fp32, bf16 or fp16 GPU tensor")
    M, K, stride = matrix_rows(torch, "x", x, kind)
    no_gradients(torch, x)
    _limits(M, K, 1)
    blocks = -(-K // BLOCK)
    codes = M * blocks * BLOCK
    # (one piece of memory for both: an allocation takes the host longer than the smallest rows take the GPU)
    rows = Fp8Rows(torch.empty(codes + M * _fours(blocks), dtype=torch.uint8, device=x.device), (0, codes), M, K,
                   made_on(x.get_device()))
    if M:
        enqueue(load_library(library), "tsplat_fp8_quantize_async", rows.index, x.data_ptr(), types[kind], stride, M, K,
                rows.codes_ptr, rows.exponents_ptr)
    return rows


def _limits(M, K, N):
    if M > MAX_ROWS or not 1 <= K <= MAX_FEATURES or not 1 <= N <= MAX_FEATURES:
        raise ValueError(f"at most {MAX_ROWS} rows and 1..{MAX_FEATURES} features in and out")


def fp8_linear(x, weight, bias=None, *, activation=None, gate=None, residual=None, out=None, out_dtype=None,
               library=None):
    """f(x8 weight^T + bias) * gate + residual, x8 the rows of x in 8 bits.

    x [..., K]: fp32, bf16 or fp16 on the GPU (unit column stride, one row stride), brought to 8 bits within the call as
    quantize_blocks does, or Fp8Rows of rows that several Linears read.  weight: Fp8Rows [N, K].  bias [N] fp32.
    activation: None or "gelu" (tanh form).  gate: fp32 [B, N] views (rows may be strided), one row for each of B equal
    runs of x's rows; residual [..., N] of the result's type.  out: None for a new tensor, residual itself, or another
    that overlaps nothing that is read.  The result has out's type, else out_dtype, else residual's, else x's (fp32 for
    Fp8Rows).  Sums are fp32.  Products are exact in results of fp32, and in calls of at most 64 rows; in bf16 and fp16
    results of more rows the 8-bit products of each 8 neighbouring values are brought to the largest one's exponent and cut
    at 2^-13 of its power of two: 2^-10 of the magnitudes that are summed at most, 1.5e-5 of a sum of random signs or so.
    Runs on torch's current stream; capturable into a HIP graph.  No gradients."""
    import torch

    types = type_ids(torch)
    if not isinstance(weight, Fp8Rows):
        raise ValueError("weight must be Fp8Rows (quantize_blocks)")
    K, N, at = weight.features, weight.rows, weight.index
    ready = isinstance(x, Fp8Rows)
    if ready:
        M, Kx, x_stride, kind, lead, x_at = x.rows, x.features, 0, torch.float32, (x.rows,), x.index
        no_gradients(torch, bias, gate, residual, out)
    else:
        kind = x.dtype if isinstance(x, torch.Tensor) else None
        if kind not in types:
            raise ValueError("x must be Fp8Rows or an fp32, bf16 or fp16 GPU tensor")
        M, Kx, x_stride = matrix_rows(torch, "x", x, kind)
        lead, x_at = x.shape[:-1], x.get_device()
        no_gradients(torch, x, bias, gate, residual, out)
    if Kx != K:
        raise ValueError(f"x has {Kx} features, the weight {K}")
    _limits(M, K, N)
    if activation not in (None, "gelu"):
        raise ValueError(f"activation is None or 'gelu', not {activation!r}")
    if bias is not None and not (isinstance(bias, torch.Tensor) and bias.dtype is torch.float32
                                 and bias.shape == (N,) and bias.is_contiguous() and bias.get_device() == at):
        raise ValueError(f"bias must be a contiguous [{N}] fp32 tensor on the GPU of the weight")
    result = next((t.dtype for t in (out, residual) if isinstance(t, torch.Tensor)), kind)
    if out_dtype is not None:
        if out is None and residual is None:
            result = out_dtype
        elif out_dtype is not result:
            raise ValueError("out_dtype is not the type of out or residual")
    if result not in types:
        raise ValueError("the result is fp32, bf16 or fp16")
    res_ptr, res_stride, gate_ptr, gate_stride, per = None, 0, None, 0, 1
    if residual is not None:
        Mr, Nr, res_stride = matrix_rows(torch, "residual", residual, result)
        if (Mr, Nr) != (M, N) or residual.get_device() != at:
            raise ValueError(f"residual must be [..., {N}] of {M} rows on the GPU of the weight")
        res_ptr = residual.data_ptr()
    if gate is not None:
        if not (isinstance(gate, torch.Tensor) and gate.dtype is torch.float32 and gate.dim() == 2
                and gate.shape[1] == N and (N == 1 or gate.stride(1) == 1) and gate.get_device() == at):
            raise ValueError(f"gate must be [B, {N}] fp32 on the GPU of the weight, with unit column stride")
        B = gate.shape[0]
        if B < 1 or M % B or (B > 1 and gate.stride(0) < N):
            raise ValueError(f"the {M} rows are not {B} equal runs, or the gate's rows overlap")
        gate_ptr, gate_stride, per = gate.data_ptr(), gate.stride(0) if B > 1 else 0, max(1, M // B)
    if out is None:
        out = torch.empty((*lead, N), dtype=result, device=weight.device)
        out_stride = N
    elif out is residual:
        out_stride = res_stride
    else:
        Mo, No, out_stride = matrix_rows(torch, "out", out, result)
        if (Mo, No) != (M, N):
            raise ValueError(f"out must be [..., {N}] of {M} rows")
    if not at == x_at == out.get_device():
        raise ValueError("x, weight and out must be on one GPU")
    if M == 0:
        return out
    for rows in (x, weight) if ready else (weight,):
        used_here(torch, rows._buffer, at, rows._stream)
    lib = load_library(library)
    need = lib.tsplat_fp8_linear_scratch_bytes(M, K, N, not ready)
    scratch = torch.empty(need, dtype=torch.uint8, device=weight.device) if need else None
    enqueue(lib, "tsplat_fp8_linear_async", at, None if ready else x.data_ptr(), types[kind], x_stride,
            x.codes_ptr if ready else None, x.exponents_ptr if ready else None,
            weight.codes_ptr, weight.exponents_ptr, bias.data_ptr() if bias is not None else None,
            int(activation is not None), gate_ptr, gate_stride, per, res_ptr, res_stride, out.data_ptr(),
            types[result], out_stride, M, K, N, scratch.data_ptr() if need else None, need)
    return out
