"""ctypes binding of libaegis_i8.so (include/aegis_i8.h): the 8-bit operators.

Operand pointers are device addresses as Python ints (``Tensor.data_ptr()``),
streams are cudaStream_t values. torch.ops.aegis.* (aegis_torch) is built on
this module. Nothing here falls back to another implementation: if the shared
library is missing, ``load()`` raises.
"""
from __future__ import annotations

import ctypes
import json
import os
from ctypes import POINTER, c_char_p, c_float, c_int, c_int64, c_size_t, c_void_p

from aegis_capi import AEGIS_OK, DTYPE_BF16, DTYPE_F16, AegisError  # noqa: F401

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "build", "libaegis_i8.so")

DTYPE_F32 = 2
MAX_K = 131071

# name -> (restype, argtypes); every function declared in include/aegis_i8.h.
_SIGNATURES = {
    "aegis_i8_last_error_string": (c_char_p, []),
    "aegis_i8_synchronize": (c_int, [c_int, c_void_p]),
    "aegis_i8_gemm": (c_int, [c_int, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_int64, c_void_p, c_int64,
                              c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_void_p, c_size_t]),
    "aegis_i8_gemm_workspace": (c_int, [c_int, c_int, c_int, c_void_p, c_int64, c_void_p, c_int64,
                                        POINTER(c_size_t)]),
    "aegis_i8_rmsnorm": (c_int, [c_int, c_void_p, c_int, c_int, c_int, c_void_p, c_int64, c_void_p, c_int64,
                                 c_void_p, c_float, c_void_p, c_int64, c_void_p, c_int64, c_void_p]),
    "aegis_i8_silu_mul": (c_int, [c_int, c_void_p, c_int, c_int, c_int, c_void_p, c_int64, c_void_p, c_int64,
                                  c_void_p, c_int64, c_void_p]),
    "aegis_i8_mlp_workspace": (c_int, [c_int, c_int, c_int, c_void_p, c_int64, c_void_p, c_int64,
                                       POINTER(c_size_t)]),
    "aegis_i8_mlp": (c_int, [c_int, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_int64, c_void_p, c_int64,
                             c_void_p, c_float, c_void_p, c_int64, c_void_p, c_void_p, c_int64, c_void_p, c_void_p,
                             c_int64, c_void_p, c_int64, c_void_p, c_size_t]),
    "aegis_i8_gemm_plan_json": (c_int, [c_int, c_int, c_int, c_int, c_char_p, c_size_t, POINTER(c_size_t)]),
}

_lib = None


def load() -> ctypes.CDLL:
    """Load libaegis_i8.so (once) and declare every C signature."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FileNotFoundError(
                f"{LIB_PATH} is not built: run `make -C aegis-core_b200` (or __graft_entry__.build())")
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def last_error_string() -> str:
    return load().aegis_i8_last_error_string().decode()


def check(status: int, where: str) -> None:
    if status != AEGIS_OK:
        raise AegisError(status, where, last_error_string())


def synchronize(device: int, stream: int) -> None:
    """Waits for `stream`; raises if a kernel's bounded wait ran out on `device` since the last check."""
    check(load().aegis_i8_synchronize(device, stream), "aegis_i8_synchronize")


def gemm_workspace(M: int, N: int, K: int, A: int, lda: int, W: int, ldw: int) -> int:
    """Bytes of workspace aegis_i8_gemm needs for these operands."""
    n = c_size_t(0)
    check(load().aegis_i8_gemm_workspace(M, N, K, A, lda, W, ldw, ctypes.byref(n)), "aegis_i8_gemm_workspace")
    return n.value


def mlp_workspace(M: int, K: int, F: int, w_gate_up: int, ld_gate_up: int, w_down: int, ld_down: int) -> int:
    """Bytes of workspace aegis_i8_mlp needs for these operands."""
    n = c_size_t(0)
    check(load().aegis_i8_mlp_workspace(M, K, F, w_gate_up, ld_gate_up, w_down, ld_down, ctypes.byref(n)),
          "aegis_i8_mlp_workspace")
    return n.value


def gemm_plan(M: int, N: int, K: int, sm_count: int = 148) -> dict:
    """The launch aegis_i8_gemm makes on a device with `sm_count` SMs (needs no GPU)."""
    buf = ctypes.create_string_buffer(512)
    needed = c_size_t(0)
    check(load().aegis_i8_gemm_plan_json(sm_count, M, N, K, buf, len(buf), ctypes.byref(needed)),
          "aegis_i8_gemm_plan_json")
    return json.loads(buf.value.decode())
