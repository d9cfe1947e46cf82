"""ctypes binding of libnsa_b200.so (the C ABI declared in include/nsa_b200.h).

There is no fallback: if the library is missing it is built with nvcc, and if that fails
the import raises.  Every wrapper raises RuntimeError with the library's own message on
a non-zero status.
"""
from __future__ import annotations

import ctypes as C
import os

import torch

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, "libnsa_b200.so")

OK = 0
ABI_VERSION = 7      # nsa_abi_version() of the library these struct mirrors and prototypes describe
BF16, FP16, FP8_E4M3, FP8_E5M2, FP32 = 0, 1, 2, 3, 4
BRANCH_COMPRESSED, BRANCH_SELECTED, BRANCH_SLIDING = 1, 2, 4
GATE_SIGMOID, GATE_SOFTMAX = 0, 1
ACTIVATIONS = {None: 0, "silu": 1, "gelu_tanh": 2, "relu": 3}
ENGINE_AUTO, ENGINE_GENERIC, ENGINE_TCGEN05 = 0, 1, 2
IO_OUT_BTHD, IO_GATES_BTHD = 1, 2

_DTYPE_CODE = {
    torch.bfloat16: BF16, torch.float16: FP16, torch.float32: FP32,
    torch.float8_e4m3fn: FP8_E4M3, torch.float8_e5m2: FP8_E5M2,
}


def dtype_code(dt: torch.dtype) -> int:
    try:
        return _DTYPE_CODE[dt]
    except KeyError:
        raise TypeError(f"unsupported dtype {dt}") from None


class FwdArgs(C.Structure):
    """Mirror of `struct nsa_fwd_args`."""
    _fields_ = [
        ("Q", C.c_void_p), ("K", C.c_void_p), ("V", C.c_void_p), ("Kc", C.c_void_p), ("Vc", C.c_void_p),
        ("idx", C.c_void_p), ("gates", C.c_void_p), ("out", C.c_void_p), ("lse", C.c_void_p),
        ("B", C.c_int32), ("H", C.c_int32), ("Hkv", C.c_int32), ("Hi", C.c_int32),
        ("Tq", C.c_int32), ("Tk", C.c_int32), ("D", C.c_int32),
        ("offset", C.c_int32),
        ("Nc", C.c_int32), ("cmp_block", C.c_int32), ("cmp_stride", C.c_int32), ("cmp_offset", C.c_int32),
        ("nq", C.c_int32), ("top_k", C.c_int32), ("bm", C.c_int32), ("bn", C.c_int32), ("sel_key_limit", C.c_int32),
        ("window", C.c_int32), ("causal", C.c_int32),
        ("branches", C.c_int32), ("fused", C.c_int32), ("gate_act", C.c_int32),
        ("q_dtype", C.c_int32), ("kv_dtype", C.c_int32), ("gate_dtype", C.c_int32),
        ("scale", C.c_float), ("q_scale", C.c_float), ("k_scale", C.c_float), ("v_scale", C.c_float),
        ("engine", C.c_int32), ("io_layout", C.c_int32),
        ("nsplit", C.c_int32), ("split_scratch", C.c_void_p), ("split_scratch_bytes", C.c_int64),
        ("dyn_len", C.c_void_p), ("accumulate", C.c_int32),
    ]


class BwdArgs(C.Structure):
    """Mirror of `struct nsa_bwd_args`."""
    _fields_ = [
        ("Q", C.c_void_p), ("K", C.c_void_p), ("V", C.c_void_p), ("dO", C.c_void_p),
        ("lse", C.c_void_p), ("delta", C.c_void_p), ("idx", C.c_void_p),
        ("dQ", C.c_void_p), ("dK_f", C.c_void_p), ("dV_f", C.c_void_p),
        ("B", C.c_int32), ("H", C.c_int32), ("Hkv", C.c_int32), ("Hi", C.c_int32),
        ("Tq", C.c_int32), ("Tk", C.c_int32), ("D", C.c_int32),
        ("nq", C.c_int32), ("top_k", C.c_int32), ("bm", C.c_int32), ("bn", C.c_int32), ("sel_key_limit", C.c_int32),
        ("offset", C.c_int32), ("causal", C.c_int32), ("dtype", C.c_int32), ("dq_dtype", C.c_int32),
        ("scale", C.c_float),
        ("branch", C.c_int32), ("window", C.c_int32),
        ("Nc", C.c_int32), ("cmp_block", C.c_int32), ("cmp_stride", C.c_int32), ("cmp_offset", C.c_int32),
        ("engine", C.c_int32), ("scratch", C.c_void_p), ("scratch_bytes", C.c_int64),
    ]


class ForwardArgs(C.Structure):
    """Mirror of `struct nsa_forward_args`."""
    _fields_ = [
        ("Q", C.c_void_p), ("K", C.c_void_p), ("V", C.c_void_p), ("gates", C.c_void_p), ("idx", C.c_void_p),
        ("out", C.c_void_p), ("ws", C.c_void_p), ("ws_bytes", C.c_int64),
        ("B", C.c_int32), ("H", C.c_int32), ("Hkv", C.c_int32), ("Hi", C.c_int32),
        ("Tq", C.c_int32), ("Tk", C.c_int32), ("D", C.c_int32),
        ("has_idx", C.c_int32), ("top_k", C.c_int32), ("force_first", C.c_int32), ("force_local", C.c_int32), ("per_group", C.c_int32),
        ("cmp_block", C.c_int32), ("cmp_stride", C.c_int32), ("bm", C.c_int32), ("bn", C.c_int32),
        ("window", C.c_int32), ("causal", C.c_int32),
        ("gate_act", C.c_int32), ("q_dtype", C.c_int32), ("gate_dtype", C.c_int32), ("engine", C.c_int32), ("io_layout", C.c_int32),
        ("scale", C.c_float), ("q_scale", C.c_float), ("k_scale", C.c_float), ("v_scale", C.c_float),
    ]


class DecodeArgs(C.Structure):
    """Mirror of `struct nsa_decode_args`."""
    _fields_ = [
        ("Q", C.c_void_p), ("K", C.c_void_p), ("V", C.c_void_p), ("Kc", C.c_void_p), ("Vc", C.c_void_p), ("Kb", C.c_void_p),
        ("gates", C.c_void_p), ("out", C.c_void_p), ("ws", C.c_void_p), ("dyn_len", C.c_void_p), ("ws_bytes", C.c_int64),
        ("B", C.c_int32), ("H", C.c_int32), ("Hkv", C.c_int32), ("Tq", C.c_int32), ("len", C.c_int32), ("D", C.c_int32),
        ("max_len", C.c_int32), ("nc_alloc", C.c_int32), ("nk_alloc", C.c_int32),
        ("cmp_block", C.c_int32), ("cmp_stride", C.c_int32), ("bm", C.c_int32), ("bn", C.c_int32), ("top_k", C.c_int32),
        ("window", C.c_int32), ("force_first", C.c_int32), ("force_local", C.c_int32), ("per_group", C.c_int32),
        ("gate_act", C.c_int32), ("dtype", C.c_int32), ("gate_dtype", C.c_int32), ("scale", C.c_float),
    ]


class NormArgs(C.Structure):
    """Mirror of `struct nsa_norm_args`."""
    _fields_ = [
        ("x", C.c_void_p), ("residual", C.c_void_p), ("weight", C.c_void_p), ("y", C.c_void_p), ("h", C.c_void_p),
        ("scale", C.c_void_p), ("rstd", C.c_void_p), ("rows", C.c_int64), ("hidden", C.c_int32),
        ("x_dtype", C.c_int32), ("res_dtype", C.c_int32), ("w_dtype", C.c_int32), ("y_dtype", C.c_int32), ("eps", C.c_float),
    ]


class NormBwdArgs(C.Structure):
    """Mirror of `struct nsa_norm_bwd_args`."""
    _fields_ = [
        ("dy", C.c_void_p), ("dh", C.c_void_p), ("h", C.c_void_p), ("weight", C.c_void_p), ("rstd", C.c_void_p),
        ("dx", C.c_void_p), ("dres", C.c_void_p), ("dweight", C.c_void_p), ("ws", C.c_void_p), ("ws_bytes", C.c_int64),
        ("rows", C.c_int64), ("hidden", C.c_int32), ("x_dtype", C.c_int32), ("res_dtype", C.c_int32), ("w_dtype", C.c_int32),
    ]


class RopeAxesArgs(C.Structure):
    """Mirror of `struct nsa_rope_axes_args`."""
    _fields_ = [
        ("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("q_out", C.c_void_p), ("k_out", C.c_void_p), ("v_out", C.c_void_p),
        ("positions", C.c_void_p), ("inv_freq", C.c_void_p),
        ("q_batch", C.c_int64), ("q_token", C.c_int64), ("k_batch", C.c_int64), ("k_token", C.c_int64), ("v_batch", C.c_int64), ("v_token", C.c_int64),
        ("B", C.c_int32), ("T", C.c_int32), ("H", C.c_int32), ("Hkv", C.c_int32), ("D", C.c_int32),
        ("n_axes", C.c_int32), ("sections", C.c_int32 * 8),
        ("pos64", C.c_int32), ("x_dtype", C.c_int32), ("y_dtype", C.c_int32), ("backward", C.c_int32),
    ]


class LinearArgs(C.Structure):
    """Mirror of `struct nsa_linear_args`."""
    _fields_ = [
        ("x", C.c_void_p), ("w", C.c_void_p), ("bias", C.c_void_p), ("residual", C.c_void_p), ("x_scale", C.c_void_p), ("w_scale", C.c_void_p),
        ("y", C.c_void_p), ("slope", C.c_void_p), ("ws", C.c_void_p), ("ws_bytes", C.c_int64),
        ("M", C.c_int32), ("N", C.c_int32), ("K", C.c_int32), ("dtype", C.c_int32), ("y_dtype", C.c_int32), ("act", C.c_int32),
    ]


class LinearBwdArgs(C.Structure):
    """Mirror of `struct nsa_linear_bwd_args`."""
    _fields_ = [
        ("dy", C.c_void_p), ("x", C.c_void_p), ("w", C.c_void_p), ("slope", C.c_void_p), ("dx", C.c_void_p), ("dw", C.c_void_p), ("dbias", C.c_void_p),
        ("ws", C.c_void_p), ("ws_bytes", C.c_int64),
        ("M", C.c_int32), ("N", C.c_int32), ("K", C.c_int32), ("dtype", C.c_int32), ("has_act", C.c_int32),
    ]


class GatedMlpArgs(C.Structure):
    """Mirror of `struct nsa_gated_mlp_args`."""
    _fields_ = [
        ("x", C.c_void_p), ("wg", C.c_void_p), ("wu", C.c_void_p), ("wd", C.c_void_p), ("residual", C.c_void_p),
        ("y", C.c_void_p), ("p", C.c_void_p), ("s", C.c_void_p), ("low", C.c_void_p), ("h", C.c_void_p), ("ws", C.c_void_p), ("ws_bytes", C.c_int64),
        ("M", C.c_int32), ("N", C.c_int32), ("F", C.c_int32), ("dtype", C.c_int32), ("act", C.c_int32),
    ]


class GatedMlpBwdArgs(C.Structure):
    """Mirror of `struct nsa_gated_mlp_bwd_args`."""
    _fields_ = [
        ("dy", C.c_void_p), ("x", C.c_void_p), ("wg", C.c_void_p), ("wu", C.c_void_p), ("wd", C.c_void_p), ("p", C.c_void_p), ("s", C.c_void_p), ("low", C.c_void_p), ("h", C.c_void_p),
        ("dx", C.c_void_p), ("dwg", C.c_void_p), ("dwu", C.c_void_p), ("dwd", C.c_void_p), ("ws", C.c_void_p), ("ws_bytes", C.c_int64),
        ("M", C.c_int32), ("N", C.c_int32), ("F", C.c_int32), ("dtype", C.c_int32),
    ]


_vp, _i, _f, _i64 = C.c_void_p, C.c_int, C.c_float, C.c_int64

PROTOTYPES = {
    "nsa_last_error": (C.c_char_p, []),
    "nsa_abi_version": (_i, []),
    "nsa_pool_mean": (_i, [_vp, _vp, _i, _i, _i, _i, _i, _i, _i, _i, _f, _vp]),
    "nsa_pool_learned": (_i, [_vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _i, _i, _vp]),
    "nsa_moba_block_indices": (_i, [_vp, _vp, _vp] + [_i] * 13 + [_f, _i, _vp]),
    "nsa_select_blocks": (_i, [_vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _i, _i, _i, _i, _i, _f, _i, _i, _i, _i, _vp]),
    "nsa_cmp_block_scores": (_i, [_vp, _vp, _vp, _vp] + [_i] * 13 + [_f, _i, _i, _i, _i, _vp]),
    "nsa_cmp_block_scores_tc": (_i, [_vp, _vp, _vp, _vp, _vp] + [_i] * 13 + [_f, _i, _i, _i, _i, _vp]),
    "nsa_topk_from_scores": (_i, [_vp, _vp, _i, _i, _i, _i, _i, _i, _i, _i, _vp]),
    "nsa_attention_fwd": (_i, [C.POINTER(FwdArgs), _vp]),
    "nsa_forward_ws_bytes": (_i64, [C.POINTER(ForwardArgs)]),
    "nsa_forward": (_i, [C.POINTER(ForwardArgs), _vp]),
    "nsa_forward_train": (_i, [C.POINTER(ForwardArgs)] + [_vp] * 6),
    "nsa_backward_ws_bytes": (_i64, [C.POINTER(ForwardArgs)]),
    "nsa_backward": (_i, [C.POINTER(ForwardArgs)] + [_vp] * 11),
    "nsa_decode_ws_bytes": (_i64, [C.POINTER(DecodeArgs)]),
    "nsa_decode": (_i, [C.POINTER(DecodeArgs), _vp]),
    "nsa_device_status": (_i, [_vp]),
    "nsa_debug_set_device_status": (_i, [_i, _i]),
    "nsa_compressed_attention_static": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _i, _i, _i, _f, _i, _vp]),
    "launch_selected_attn_fwd": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _i, _i, _f, _vp]),
    "nsa_bwd_delta": (_i, [_vp, _vp, _vp, _i64, _i, _i, _vp]),
    "nsa_selected_bwd": (_i, [C.POINTER(BwdArgs), _vp]),
    "nsa_attention_bwd": (_i, [C.POINTER(BwdArgs), _vp]),
    "nsa_attention_bwd_scratch_bytes": (_i64, [C.POINTER(BwdArgs)]),
    "nsa_pool_mean_bwd": (_i, [_vp, _vp, _i, _i, _i, _i, _i, _i, _i, _vp]),
    "launch_selected_attn_bwd": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _i, _i, _f, _vp]),
    "nsa_combine": (_i, [_vp, _vp, _vp, _vp, _vp, _i64, _i, _i, _i, _i, _vp]),
    "nsa_fp8_absmax": (_i, [_vp, _i64, _i, _vp, _vp]),
    "nsa_fp8_quantize": (_i, [_vp, _vp, _i64, _i, _i, _f, _vp]),
    "nsa_fp8_dequantize": (_i, [_vp, _vp, _i64, _i, _f, _vp]),
    "nsa_cast_from_f32": (_i, [_vp, _vp, _i64, _i, _vp]),
    "nsa_rope_to_heads": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _i, _vp]),
    "nsa_cache_append": (_i, [_vp] * 7 + [_i] * 12 + [_vp]),
    "nsa_cache_append_dev": (_i, [_vp] * 7 + [_i] * 4 + [_vp] + [_i] * 7 + [_vp]),
    "nsa_select_blocks_cached": (_i, [_vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _i, _i, _i, _vp, _f, _i, _i, _i, _i, _vp]),
    "nsa_rms_norm": (_i, [C.POINTER(NormArgs), _vp]),
    "nsa_rms_norm_bwd_ws_bytes": (_i64, [_i64, _i]),
    "nsa_rms_norm_bwd": (_i, [C.POINTER(NormBwdArgs), _vp]),
    "nsa_quantize_rows_fp8": (_i, [_vp, _vp, _vp, _i64, _i, _i, _i, _vp]),
    "nsa_rope_axes": (_i, [C.POINTER(RopeAxesArgs), _vp]),
    "nsa_linear_ws_bytes": (_i64, [C.POINTER(LinearArgs)]),
    "nsa_linear": (_i, [C.POINTER(LinearArgs), _vp]),
    "nsa_linear_bwd_ws_bytes": (_i64, [C.POINTER(LinearBwdArgs)]),
    "nsa_linear_bwd": (_i, [C.POINTER(LinearBwdArgs), _vp]),
    "nsa_gated_mlp_ws_bytes": (_i64, [C.POINTER(GatedMlpArgs)]),
    "nsa_gated_mlp": (_i, [C.POINTER(GatedMlpArgs), _vp]),
    "nsa_gated_mlp_bwd_ws_bytes": (_i64, [C.POINTER(GatedMlpBwdArgs)]),
    "nsa_gated_mlp_bwd": (_i, [C.POINTER(GatedMlpBwdArgs), _vp]),
    "nsa_memcpy_2d": (_i, [_vp, C.c_size_t, _vp, C.c_size_t, C.c_size_t, C.c_size_t, _i, _vp]),
}

_lib = None


def load() -> C.CDLL:
    """Load (building first if needed) the shared library; raises if that is impossible."""
    global _lib
    if _lib is not None:
        return _lib
    from . import build as _build
    try:
        _build.build()               # returns at once when the stamp of the source hashes matches the built library
    except RuntimeError:
        if not os.path.exists(LIB_PATH):
            raise                    # nothing to load; with a library present (no nvcc on this machine) the ABI check decides
    lib = C.CDLL(LIB_PATH)
    for name, (res, args) in PROTOTYPES.items():
        fn = getattr(lib, name)      # AttributeError if the symbol is missing
        fn.restype, fn.argtypes = res, args
    if lib.nsa_abi_version() != ABI_VERSION:
        raise RuntimeError(f"{LIB_PATH} has ABI version {lib.nsa_abi_version()}, this package expects {ABI_VERSION}: "
                           "rebuild with `python -m nsa_from_scratch_b200.build --force`")
    _lib = lib
    return lib


_torch_ops = None


def torch_ops():
    """The compiled torch side of the layer's operators (built first if needed); raises if that is impossible."""
    global _torch_ops
    if _torch_ops is None:
        from . import build as _build
        load()                       # checks the ABI version of the library that the module links to
        try:
            path = _build.build_torch()
        except _build.NoCompiler:    # a source that does not compile is an error, whatever was built before it
            path = _build.TORCH_LIB
            if not os.path.exists(path):
                raise                # with a module present the checks below decide
        import importlib.util
        spec = importlib.util.spec_from_file_location("_nsa_torch", path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        built = getattr(module, "abi_version", None)
        if built != ABI_VERSION:
            raise RuntimeError(f"{path} was built for ABI version {built}, this package expects {ABI_VERSION}: "
                               "rebuild with `python -m nsa_from_scratch_b200.build --force`")
        _torch_ops = module
    return _torch_ops


def check(rc: int, what: str) -> None:
    if rc != OK:
        msg = load().nsa_last_error().decode("utf-8", "replace")
        raise RuntimeError(f"{what} failed (status {rc}): {msg}")


def stream_ptr(device=None) -> int:
    if device is None:
        return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())   # no Stream object on the way
    return torch.cuda.current_stream(device).cuda_stream


class _NoGuard:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_NO_GUARD = _NoGuard()


def on_device(t):
    """Context in which `t`'s device is current.  Almost every call finds it current already, and entering
    torch.cuda.device costs several microseconds of a short launch."""
    return _NO_GUARD if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def ptr(t) -> int:
    return 0 if t is None else t.data_ptr()
