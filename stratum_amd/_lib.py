"""ctypes binding of libstratum_nf4.so (the C ABI declared in include/stratum_nf4.h).

torch is imported first on purpose: torch ships its own HIP runtime with the
same SONAME (libamdhip64.so.7), so loading the library after torch binds it to
that runtime and torch's streams and device pointers are valid handles for it.
There is no fallback: if the library is missing every call raises.
"""

from __future__ import annotations

import contextlib
import ctypes
import functools
import os
import threading

import torch  # noqa: F401  (must be loaded before the HIP library, see above)

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(PKG_DIR, "libstratum_nf4.so")

STM_OK = 0
STM_ERR_INVALID = -1
STM_ERR_UNSUPPORTED = -2
STM_ERR_HIP = -3

STM_F16, STM_BF16, STM_F32 = 0, 1, 2
STM_NF4_ARGMIN, STM_NF4_THRESHOLD = 0, 1

ABI_VERSION = 5

# (name, argtypes) of every entry point of include/stratum_nf4.h
_P = ctypes.c_void_p
_I64 = ctypes.c_int64
_I = ctypes.c_int
_D = ctypes.c_double
SIGNATURES = {
    "stm_nf4_abi_version": ([], _I),
    "stm_last_error": ([], ctypes.c_char_p),
    "stm_nf4_quantize": ([_P, _I, _I64, _I, _I, _P, _P, _P], _I),
    "stm_nf4_dequantize": ([_P, _P, _I64, _I, _P, _I, _P], _I),
    "stm_nf4_gemm_fwd": ([_P, _P, _P, _P, _P, _P, _I, _P, _I64, _I64, _I64, _I, _I, _P, _I64, _P], _I),
    "stm_nf4_gemm_bwd_dx": ([_P, _P, _P, _P, _P, _I, _P, _I64, _I64, _I64, _I, _I, _P, _I64, _P], _I),
    "stm_nf4_gemm_workspace_bytes": ([_I64, _I64, _I64, _I], _I64),
    "stm_nf4_gemm_fwd_noalloc": ([_P, _P, _P, _P, _P, _P, _I, _P, _I64, _I64, _I64, _I, _I, _P], _I),
    "stm_nf4_gemm_set_tile": ([_I], _I),
    "stm_nf4_grouped_gemm_fwd": ([_P, _P, _P, _P, _P, _I, _I64, _P, _I64, _I64, _I, _I, _P], _I),
    "stm_nf4_grouped_tile_rows": ([_P, _I], _I),
    "stm_nf4_quantize_many": ([_I, _P, _P, _I, _I, _I, _P, _P, _P], _I),
    "stm_nf4_dequantize_many": ([_I, _P, _P, _P, _I, _P, _I, _P], _I),
    "stm_nf4_dequantize_host": ([_I, _P, _P, _P, _I, _P, _I, _P], _I),
    "stm_event_done": ([_P], _I),
    "stm_nf4_grouped_gemm_bwd_dx": ([_P, _P, _P, _P, _P, _I, _I64, _P, _I64, _I64, _I, _I, _P], _I),
    "stm_swiglu_fwd": ([_P, _P, _I64, _I64, _I, _P], _I),
    "stm_swiglu_bwd": ([_P, _P, _P, _I64, _I64, _I, _P], _I),
    "stm_nf4_gated_workspace_bytes": ([_I64, _I64, _I64], _I64),
    "stm_nf4_gated_keep_workspace_bytes": ([_I64, _I64, _I64], _I64),
    "stm_nf4_gated_fwd": ([_P, _P, _P, _P, _I64, _I64, _I64, _I, _I, _P, _I64, _P], _I),
    "stm_nf4_gated_bwd": ([_P, _P, _P, _P, _P, _I64, _I64, _I64, _I, _I, _P, _I64, _P], _I),
    "stm_nf4_gated_sums_bytes": ([_I64, _I64, _I64], _I64),
    "stm_nf4_gated_fwd_keep": ([_P, _P, _P, _P, _P, _I64, _I64, _I64, _I, _I, _P, _I64, _P], _I),
    "stm_gated_bwd_kept": ([_P, _P, _P, _I64, _I64, _I, _P], _I),
    "stm_lora_workspace_bytes": ([_I64, _I64, _I, _I], _I64),
    "stm_lora_down": ([_P, _P, _P, _I64, _I64, _I, ctypes.c_float, _I, _P, _I64, _P], _I),
    "stm_lora_dy": ([_P, _P, _P, _P, _P, _I64, _I64, _I, ctypes.c_float, _I, _P, _I64, _P], _I),
    "stm_lora_down_aug": ([_P, _P, _P, _P, _I64, _I64, _I, ctypes.c_float, _I, _P, _I64, _P], _I),
    "stm_nf4_dequantize_aug": ([_P, _P, _P, _I, _P, _I64, _I64, _I, _I, _P], _I),
    "stm_lora_up": ([_P, _P, _P, _P, _I64, _I64, _I, _I, _I, _P], _I),
    "stm_lora_da": ([_P, _P, _P, _I64, _I64, _I, _I, _P, _I64, _P], _I),
    "stm_grad_norm_workspace_bytes": ([_I, _P], _I64),
    "stm_grad_norm": ([_I, _P, _P, _I, _D, _D, _P, _P, _I64, _P], _I),
    "stm_adamw_step": ([_I, _P, _I, _I, _I, _D, _D, _D, _D, _D, _I64, _P, _P], _I),
    "stm_adamw_table_bytes": ([_I], _I64),
    "stm_adamw_fill_table": ([_I, _P, _I, _I, _I, _P], _I),
    "stm_adamw_step_table": ([_I, _P, _I, _I, _I, _I, _D, _D, _D, _D, _D, _I64, _P, _P], _I),
    "stm_state8_codes": ([_P, _I64, _I, _P, _P, _P], _I),
    "stm_state8_values": ([_P, _P, _I64, _I, _P, _P], _I),
    "stm_rms_norm_fwd": ([_P, _P, _I, _P, _I, _P, _P, _P, _I64, _I64, _D, _I, _P], _I),
    "stm_rms_norm_workspace_bytes": ([_I64, _I64], _I64),
    "stm_rms_norm_bwd": ([_P, _P, _P, _P, _I, _P, _P, _I, _P, _P, _P, _I64, _I64, _I, _P, _I64, _P], _I),
    "stm_moe_route": ([_P, _P, _P, _P, _P, _I64, _I, _I, _I, _I, _I, _I, _I, _D, _I, _P], _I),
    "stm_moe_route_bwd": ([_P, _P, _P, _P, _I64, _I, _I, _I, _I, _D, _I, _P], _I),
    "stm_moe_sort_workspace_bytes": ([_I64, _I], _I64),
    "stm_moe_sort": ([_P, _I64, _I, _P, _P, _P, _P, _I64, _P], _I),
    "stm_moe_gather": ([_P, _P, _P, _I, _P, _I64, _I, _I64, _I, _P], _I),
    "stm_moe_combine": ([_P, _I64, _P, _P, _P, _P, _I, _I64, _I, _I64, _I, _P], _I),
    "stm_moe_combine_bwd": ([_P, _I, _P, _I64, _P, _P, _P, _I, _P, _P, _I64, _I, _I64, _I, _P], _I),
    "stm_nf4_decision_boundaries": ([_I, _P], _I),
    "stm_nf4_cell_table": ([_I, _P, _P], _I),
}


class NF4LibraryError(RuntimeError):
    """The HIP library is missing or failed to load."""


class NF4KernelError(RuntimeError):
    """A library entry point returned a non-zero status."""

    def __init__(self, what: str, code: int, reason: str):
        super().__init__(f"{what} failed (status {code}): {reason}")
        self.code = code
        self.reason = reason


_lib = None
_lock = threading.Lock()


def lib():
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise NF4LibraryError(
                    f"{LIB_PATH} is not built; build it with `python -m stratum_amd._build` "
                    "(or __graft_entry__.build())")
            try:
                L = ctypes.CDLL(LIB_PATH)
            except OSError as exc:
                raise NF4LibraryError(f"cannot load {LIB_PATH}: {exc}") from exc
            for name, (args, res) in SIGNATURES.items():
                fn = getattr(L, name)
                fn.argtypes = args
                fn.restype = res
            if L.stm_nf4_abi_version() != ABI_VERSION:
                raise NF4LibraryError(f"ABI version {L.stm_nf4_abi_version()} != {ABI_VERSION}")
            _lib = L
    return _lib


_fast = None


def fast():
    """The native host code of launch-bound calls (csrc/fast_path.cpp)."""
    global _fast
    if _fast is None:
        try:
            from . import _fast as module
        except ImportError as exc:
            raise NF4LibraryError(f"{PKG_DIR}/_fast.so is not built or does not load ({exc}); build it with "
                                  "`python -m stratum_amd._build` (or __graft_entry__.build())") from exc
        _fast = module
    return _fast


_SPARSE = ("stm_last_error", "stm_rms_norm_fwd", "stm_rms_norm_workspace_bytes", "stm_rms_norm_bwd", "stm_moe_route",
           "stm_moe_route_bwd", "stm_moe_sort_workspace_bytes", "stm_moe_sort", "stm_moe_gather", "stm_moe_combine",
           "stm_moe_combine_bwd")
_sparse = None


def sparse():
    """:func:`fast` with the entry points that csrc/sparse_path.cpp calls."""
    global _sparse
    if _sparse is None:
        module = fast()
        module.sparse_setup([address(name) for name in _SPARSE])
        _sparse = module
    return _sparse


def taken(what: str, out):
    """*out* of a native call that was given checked operands."""
    if out is None:
        raise RuntimeError(f"{what}: the native host code does not take these operands")
    return out


@functools.lru_cache(maxsize=None)
def address(name: str) -> int:
    """Address of an entry point, for native callers."""
    return ctypes.cast(getattr(lib(), name), ctypes.c_void_p).value


def check(rc: int, what: str) -> None:
    if rc != STM_OK:
        reason = (lib().stm_last_error() or b"").decode(errors="replace")
        if rc in (STM_ERR_INVALID, STM_ERR_UNSUPPORTED):
            raise ValueError(f"{what}: {reason} (status {rc})")
        raise NF4KernelError(what, rc, reason)


def dtype_tag(dtype: torch.dtype) -> int:
    if dtype == torch.float16:
        return STM_F16
    if dtype == torch.bfloat16:
        return STM_BF16
    if dtype == torch.float32:
        return STM_F32
    raise ValueError(f"unsupported dtype {dtype} (expected float16, bfloat16 or float32)")


def _index(device: torch.device) -> int:
    return torch.cuda.current_device() if device.index is None else device.index


def stream_handle(device: torch.device) -> int:
    """hipStream_t of torch's current stream on *device* (the handle alone: a
    ``torch.cuda.Stream`` object costs 1.7 us more)."""
    return torch._C._cuda_getCurrentRawStream(_index(device))


_SAME_DEVICE = contextlib.nullcontext()


def device_guard(device: torch.device):
    """``torch.cuda.device(device)``, or nothing where it is the current device
    already (every call of a one-process-per-GPU program: 1.2 us each)."""
    return _SAME_DEVICE if torch.cuda.current_device() == device.index else torch.cuda.device(device)
