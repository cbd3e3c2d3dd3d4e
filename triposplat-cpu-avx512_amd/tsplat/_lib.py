"""Loader for libtsplat_hip.so (gfx950 kernels behind a C ABI).

torch is imported before the library is opened so that the HIP runtime torch
already loaded (SONAME libamdhip64.so.7) is the one the library binds to.
There is no fallback: if the library is missing, every entry point raises.
"""
from __future__ import annotations

import ctypes
import os
from pathlib import Path

PACKAGE_DIR = Path(__file__).resolve().parent
DEFAULT_LIBRARY = PACKAGE_DIR / "lib" / "libtsplat_hip.so"

_vp = ctypes.c_void_p
_i = ctypes.c_int
_i64 = ctypes.c_int64

# name -> (argtypes, restype); the C declarations are in include/tsplat_hip.h.
SIGNATURES = {
    "triposplat_gemm_rnf8_avx512": ([_vp] * 10 + [_i] * 7, _i),
    "triposplat_gemm_rnf8_avx512_range": ([_vp] * 10 + [_i] * 9, _i),
    "triposplat_gemm_rnf8_avx512_tail": ([_vp] * 10 + [_i] * 7, _i),
    "triposplat_gemm_rnf8_avx512_row_tile": ([], _i),
    "triposplat_gemm_rnf8_avx512_residual_mode": ([], _i),
    "tsplat_nf24_gemm_async": ([_vp] * 6 + [_i] * 7 + [_vp], _i),
    "triposplat_sdpa_f32_avx512_exact_q8t512": ([_vp] * 5 + [_i] * 8, _i),
    "triposplat_sdpa_f32": ([_vp] * 5 + [_i] * 8, _i),
    "triposplat_sdpa_f32_avx512_exact_q8": ([_vp] * 5 + [_i] * 8, _i),
    "triposplat_sdpa_f32_avx512_exact_q8t512_packed_blhd": ([_vp] * 5 + [_i] * 9, _i),
    "triposplat_sdpa_key_tile": ([], _i),
    "triposplat_sdpa_query_block": ([], _i),
    "triposplat_sdpa_packed_output_is_blhd": ([], _i),
    "triposplat_sdpa_q8t512_profile_reset": ([], None),
    "triposplat_sdpa_q8t512_profile_get": ([ctypes.POINTER(ctypes.c_uint64)] * 5, _i),
    "triposplat_sdpa_q8t512_workspace_stats": ([ctypes.POINTER(ctypes.c_uint64)] * 2, _i),
    "triposplat_sdpa_q8t512_workspace_release": ([], None),
    "tsplat_sdpa_async": ([_vp] * 5 + [_i] * 7 + [_i64] + [_i] * 3 + [_vp], _i),
    "tsplat_sdpa_precision_async": ([_vp] * 5 + [_i] * 7 + [_i64] + [_i] * 4 + [_vp], _i),
    "tsplat_sdpa_noalloc_async": ([_vp] * 5 + [_i] * 7 + [_i64] + [_i] * 4 + [_vp], _i),
    "triposplat_qkv_rope_rmsnorm_pack_f32_avx512_v2": ([_vp] * 7 + [_i] * 7, _i),
    "triposplat_qkv_rope_rmsnorm_pack_f32_avx512": ([_vp] * 7 + [_i] * 7, _i),
    "triposplat_qkv_postprocess_token_tile": ([], _i),
    "triposplat_qkv_postprocess_v2_tail_only_clear": ([], _i),
    "triposplat_qkv_postprocess_bf16_probe_mode": ([], _i),
    "triposplat_gemm_nf24_qkv_rope_rmsnorm_pack_f32_avx512": ([_vp] * 15 + [_i] * 10, _i),
    "triposplat_gemm_nf24_qkv_direct_row_tile": ([], _i),
    "triposplat_gemm_nf24_qkv_direct_tile_bytes": ([], _i),
    "triposplat_gemm_nf24_qkv_direct_residual_mode": ([], _i),
    "triposplat_q_kv_selected_rope_rmsnorm_pack_f32_avx512_v2": ([_vp] * 9 + [_i] * 8, _i),
    "tsplat_q_kv_selected_postprocess_async": ([_vp] * 9 + [_i] * 8 + [_vp], _i),
    "tsplat_qkv_postprocess_async": ([_vp] * 7 + [_i] * 7 + [_vp], _i),
    "tsplat_gemm_nf24_qkv_direct_async": ([_vp] * 11 + [_i] * 8 + [_vp], _i),
    "tsplat_gemm_nf24_qkv_direct_ex_async": ([_vp] * 11 + [_i] * 11 + [_vp], _i),
    "tsplat_nf24_pack_async": ([_vp, _i, _i, _vp, _i, _vp, _vp, _vp, _vp, _vp], _i),
    "tsplat_nf24_pack_stats_bytes": ([_i, _i], _i64),
    "tsplat_nf24_pack_stats_async": ([_vp, _i, _i, _vp, _i, _vp, _vp, _vp, _vp, _vp, _vp], _i),
    "tsplat_nf24_decode_async": ([_vp] * 4 + [_i] * 3 + [_vp], _i),
    "tsplat_nf24_gemm_epilogue_async": ([_vp] * 6 + [_i] * 8 + [_vp, _i64, _i, _vp], _i),
    "tsplat_nf24_gemm_precision_async": ([_vp] * 6 + [_i] * 8 + [_vp, _i64, _i, _i, _vp], _i),
    "tsplat_nf24_gemm_planes_async": ([_vp] * 6 + [_i] * 8 + [_vp, _i64, _i, _i, _vp, _vp, _vp], _i),
    "tsplat_nf24_bf16_planes_async": ([_vp] * 3 + [_i] * 3 + [_vp] * 3, _i),
    "tsplat_gemm_nf24_qkv_direct_planes_async": ([_vp] * 11 + [_i] * 11 + [_vp] * 3, _i),
    "triposplat_layernorm_f32_avx512": ([_vp] * 4 + [_i64, _i, ctypes.c_float, _i, _i], _i),
    "triposplat_multihead_rmsnorm_f32_avx512": ([_vp] * 3 + [_i64, _i, _i, ctypes.c_float, _i], _i),
    "triposplat_rope_complex_f32_avx512": ([_vp] * 3 + [_i64, _i, _i], _i),
    "triposplat_modulate_inplace_f32_avx512": ([_vp] * 3 + [_i] * 4, _i),
    "triposplat_gated_residual_inplace_f32_avx512": ([_vp] * 3 + [_i] * 4, _i),
    "triposplat_add_inplace_f32_avx512": ([_vp] * 2 + [_i64, _i], _i),
    "triposplat_gelu_tanh_f32_avx512": ([_vp] * 2 + [_i64, _i], _i),
    "triposplat_silu_f32_avx512": ([_vp] * 2 + [_i64, _i], _i),
    "triposplat_cfg_combine_inplace_f32_avx512": ([_vp] * 3 + [_i, _i64, _i], _i),
    "triposplat_euler_update_inplace_f32_avx512": ([_vp] * 3 + [_i, _i64, _i], _i),
    "triposplat_ab2_update_inplace_f32_avx512": ([_vp] * 5 + [_i, _i64, _i], _i),
    "tsplat_layernorm_modulate_async": ([_vp] * 4 + [_i64, _i, ctypes.c_float, _i, _vp, _vp, _i64,
                                         _i64, _vp], _i),
    "tsplat_head_rmsnorm_async": ([_vp, _i64, _vp, _vp] + [_i] * 4 + [ctypes.c_float, _i, _i, _vp], _i),
    "tsplat_rope_complex_async": ([_vp] * 3 + [_i64, _i, _vp], _i),
    "tsplat_modulate_async": ([_vp] * 3 + [_i] * 3 + [_vp], _i),
    "tsplat_gated_residual_async": ([_vp] * 3 + [_i] * 3 + [_vp], _i),
    "tsplat_add_async": ([_vp] * 2 + [_i64, _vp], _i),
    "tsplat_gelu_tanh_async": ([_vp] * 2 + [_i64, _vp], _i),
    "tsplat_silu_async": ([_vp] * 2 + [_i64, _vp], _i),
    "tsplat_cfg_combine_async": ([_vp] * 3 + [_i, _i64, _vp], _i),
    "tsplat_euler_update_async": ([_vp] * 3 + [_i, _i64, _vp], _i),
    "tsplat_ab2_update_async": ([_vp] * 5 + [_i, _i64, _vp], _i),
    "tsplat_abi_version": ([], _i),
    "tsplat_last_hip_error": ([], _i),
    "tsplat_build_arch": ([], ctypes.c_char_p),
}

# The operators that serve a batch of several requests; declared in
# include/tsplat_hip_requests.h, with a version of their own.
REQUEST_SIGNATURES = {
    "tsplat_requests_abi_version": ([], _i),
    "tsplat_low_rank_scratch_bytes": ([_i] * 6, _i64),
    "tsplat_low_rank_add_async": ([_vp, _i64, _vp, _i64] + [_vp] * 6 + [_i64] + [_i] * 6 + [_vp, _i64, _vp], _i),
    "tsplat_residual_norm_async": ([_vp, _i64] * 4 + [_i64, _i, ctypes.c_float, _vp, _i64]
                                   + [_i, _vp, _vp, ctypes.c_float] * 2 + [_vp, _vp, _i64, _i64, _vp], _i),
    "tsplat_rope_axes_async": ([_vp] + [_i64] * 4 + [_i] + [_vp] * 6 + [_i] * 3 + [_vp] * 2
                               + [_i, ctypes.c_float] + [_i] * 5 + [_vp], _i),
}

STATUS_TEXT = {
    -1: "null pointer",
    -2: "bad sizes / stages / head dim",
    -3: "range, stride or key-bias length mismatch",
    -4: "range not 16-aligned or pointer not 16-byte aligned",
    -5: "device workspace allocation failed",
    -6: "not device memory of the current device, or allocation too small",
    -7: "HIP launch / runtime error",
    -8: "needs more scratch than the no-allocation entry point's static buffer",
}

# tsplat_abi_version() of the library these bindings describe: it moves
# whenever an entry's argument list changes (ABI 3 put kv_round before the
# stream argument of the asynchronous QKV entries: a library reporting another
# version would read its arguments shifted) or entries are added (ABI 4: the
# bf16 weight planes; ABI 5: the packer's error figures).
ABI_VERSION = 5
# tsplat_requests_abi_version(), likewise, of REQUEST_SIGNATURES.
REQUESTS_ABI_VERSION = 1

_CACHE: dict[str | None, ctypes.CDLL] = {}  # by resolved name; None: DEFAULT_LIBRARY, which needs no resolving


def library_path(path: str | os.PathLike | None = None) -> Path:
    if path is not None:
        return Path(path).resolve()
    env = os.environ.get("TSPLAT_HIP_LIBRARY")
    return Path(env).resolve() if env else DEFAULT_LIBRARY


def load_library(path: str | os.PathLike | None = None) -> ctypes.CDLL:
    """Open libtsplat_hip.so once per path and set every argtypes/restype."""
    # without a name there is nothing to resolve: small calls are bound by the host, and the look at the file system
    # would take longer than the rest of them
    unnamed = path is None and not os.environ.get("TSPLAT_HIP_LIBRARY")
    lib = _CACHE.get(None) if unnamed else None
    if lib is not None:
        return lib
    import torch  # noqa: F401  (binds the library to torch's HIP runtime)

    resolved = library_path(path)
    key = resolved.as_posix()
    lib = _CACHE.get(key)
    if lib is not None:
        if unnamed:
            _CACHE[None] = lib
        return lib
    if not resolved.is_file():
        raise FileNotFoundError(
            f"libtsplat_hip.so not found at {resolved}; build it with "
            "`make -C triposplat-cpu-avx512_amd` (there is no CPU fallback)"
        )
    lib = ctypes.CDLL(key)
    for name, (argtypes, restype) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.argtypes = argtypes
        fn.restype = restype
    found = lib.tsplat_abi_version()
    if found != ABI_VERSION:
        raise RuntimeError(
            f"{resolved} reports ABI version {found}, these bindings expect {ABI_VERSION}; "
            "rebuild it with `make -C triposplat-cpu-avx512_amd`"
        )
    for name, (argtypes, restype) in REQUEST_SIGNATURES.items():
        fn = getattr(lib, name, None)
        if fn is None:
            raise RuntimeError(f"{resolved} has no {name}; rebuild it with `make -C triposplat-cpu-avx512_amd`")
        fn.argtypes = argtypes
        fn.restype = restype
    found = lib.tsplat_requests_abi_version()
    if found != REQUESTS_ABI_VERSION:
        raise RuntimeError(
            f"{resolved} reports version {found} of its request operators, these bindings expect "
            f"{REQUESTS_ABI_VERSION}; rebuild it with `make -C triposplat-cpu-avx512_amd`"
        )
    _CACHE[key] = lib
    return lib


def check_status(status: int, what: str) -> None:
    if status != 0:
        raise RuntimeError(f"{what} returned status {status} ({STATUS_TEXT.get(status, 'unknown')})")


def current_stream_handle(device) -> int:
    """Raw hipStream_t of torch's current stream on `device`."""
    import torch

    return int(torch.cuda.current_stream(device).cuda_stream)


# ---- shared by the wrappers of REQUEST_SIGNATURES.  Small calls are bound by the host, a microsecond for every few
# attribute reads: these take each fact about a tensor once.
_RAW_STREAM = None


def _raw_stream(index: int) -> int:
    """hipStream_t of torch's current stream on device `index`, without building a torch.cuda.Stream (1.8 us)."""
    global _RAW_STREAM
    if _RAW_STREAM is None:
        import torch

        _RAW_STREAM = getattr(torch._C, "_cuda_getCurrentRawStream", None) or current_stream_handle
    return _RAW_STREAM(index)


def enqueue(lib, fn_name, index, *args) -> None:
    """Calls an asynchronous entry on torch's current stream of device `index`; raises on a nonzero status."""
    import torch

    stream = _raw_stream(index)
    if torch.cuda.current_device() == index:
        status = getattr(lib, fn_name)(*args, stream)
    else:
        with torch.cuda.device(index):
            status = getattr(lib, fn_name)(*args, stream)
    if status != 0:
        check_status(status, fn_name)


def no_gradients(torch, *tensors) -> None:
    """These operators have no backward and no forward mode: a tensor that expects a gradient or carries a tangent is
    refused, not cut off in silence."""
    forward = torch.autograd.forward_ad
    duals = getattr(forward, "_current_level", 0) >= 0  # (outside of a dual level no tensor has a tangent)
    for t in tensors:
        if t is not None and (t.requires_grad and torch.is_grad_enabled()
                              or duals and forward.unpack_dual(t).tangent is not None):
            raise ValueError("this operator has no backward or forward mode of gradients: call it under "
                             "torch.no_grad() and outside of dual levels, or detach its inputs")


def rows_of(torch, name, t, cols) -> tuple[int, int]:
    """(rows, row stride) of a GPU fp32 tensor [..., cols] whose rows lie at one stride; ValueError otherwise."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype is torch.float32):
        raise ValueError(f"{name} must be an fp32 GPU tensor")
    shape = t.shape
    if len(shape) == 0 or shape[-1] != cols:
        raise ValueError(f"{name} must have {cols} columns, its shape is {list(shape)}")
    if t.is_contiguous():
        return t.numel() // cols, cols
    steps = t.stride()
    if cols > 1 and steps[-1] != 1:
        raise ValueError(f"{name} must have unit column stride")
    rows, stride = 1, None
    for size, step in zip(reversed(shape[:-1]), reversed(steps[:-1])):
        if size != 1:
            if stride is None:
                stride = step
            elif step != stride * rows:
                raise ValueError(f"the rows of {name} must lie at one stride")
            rows *= size
    if stride is not None and rows > 1 and stride < cols:
        raise ValueError(f"the rows of {name} overlap")
    return rows, cols if stride is None else stride
