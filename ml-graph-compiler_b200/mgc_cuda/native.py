"""The libmgc_cuda C ABI bound with ctypes: library loading, signatures, status checks.

What ``include/mgc_cuda.h`` declares, without the compiler half of the package: the kernel ABI
works on device pointers and needs no reference compiler (the binding of
``codegen/runtime_lib.py:59-68``).
"""

from __future__ import annotations

import ctypes
import threading
from pathlib import Path
from typing import Any

from mgc_cuda import build as _build
from mgc_cuda._errors import CodegenError, GraphError

_LIB: ctypes.CDLL | None = None
_LIB_LOCK = threading.Lock()

# Every symbol include/mgc_cuda.h declares, with its ctypes signature.
_VP, _I, _I64, _F, _D = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_double
SIGNATURES: dict[str, tuple[Any, list[Any]]] = {
    "mgc_cuda_abi_version": (_I, []),
    "mgc_cuda_last_error": (ctypes.c_char_p, []),
    "mgc_cuda_device_supported": (_I, [_I]),
    "mgc_cuda_create": (_I, [_VP, _I, _VP, _I64, _VP, _I64, _I64, _I64, _VP, _I, _VP, _I, _I, ctypes.POINTER(_VP)]),
    "mgc_cuda_run": (_I, [_VP, _VP, _VP]),
    "mgc_cuda_run_device": (_I, [_VP, _I]),
    "mgc_cuda_set_input_chunks": (_I, [_VP, _I, _I, _I64, _VP, _I]),
    "mgc_cuda_input_ptr": (_VP, [_VP, _I]),
    "mgc_cuda_output_ptr": (_VP, [_VP, _I]),
    "mgc_cuda_stream": (_VP, [_VP]),
    "mgc_cuda_profile": (_I, [_VP, ctypes.POINTER(_D), _I]),
    "mgc_cuda_launch_count": (_I, [_VP]),
    "mgc_cuda_gemm_paths": (_I, [_VP, ctypes.POINTER(ctypes.c_int32), _I]),
    "mgc_cuda_arena_bytes": (_I64, [_VP]),
    "mgc_cuda_weights_bytes": (_I64, [_VP]),
    "mgc_cuda_destroy": (None, [_VP]),
    "mgc_cuda_execute": (_I, [_VP, _I, _VP, _I64, _VP, _VP]),
    "mgc_cuda_gemm": (
        _I,
        [_I, _I, _I, _I, _VP, _I64, _I64, _I64, _VP, _I64, _I64, _I64, _VP, _I64, _I64, _F, _VP, _I, _VP,
         _I64, _I64, _F, _I, _F, _F, _I, _VP],
    ),
    "mgc_cuda_conv_nhwc": (
        _I,
        [_I] * 15 + [_VP, _VP, _VP, _VP, _I, _F, _F, _VP, _I, _VP],
    ),
    "mgc_cuda_conv_nhwc_noalloc": (_I, [_I] * 15 + [_VP, _VP, _VP, _VP, _I, _F, _F, _VP, _VP]),
    "mgc_cuda_depthwise_nhwc": (_I, [_I] * 14 + [_VP, _VP, _VP, _VP, _I, _F, _F, _VP, _VP]),
    "mgc_cuda_pool_nhwc": (_I, [_I] * 18 + [_VP, _VP, _VP]),
    "mgc_cuda_reduce_mid": (_I, [_I, _I64, _I64, _I64, _VP, _VP, _VP]),
    "mgc_cuda_softmax": (_I, [_I64, _I64, _I64, _VP, _VP, _I, _VP]),
    "mgc_cuda_layer_norm": (_I, [_I64, _I64, _VP, _VP, _VP, _F, _VP, _VP]),
    "mgc_cuda_kv_append": (_I, [_VP, _VP]),
    "mgc_cuda_paged_attention": (_I, [_VP, _VP]),
    "mgc_cuda_paged_attention_workspace": (_I64, [_VP]),
    "mgc_cuda_kv_append_heads": (_I, [_VP, _VP]),
    "mgc_cuda_kv_read": (_I, [_VP, _VP]),
    "mgc_cuda_paged_attention_quantized": (_I, [_VP, _VP]),
    "mgc_cuda_paged_attention_quantized_workspace": (_I64, [_VP]),
}


def library(path: str | Path | None = None) -> ctypes.CDLL:
    """Load libmgc_cuda.so (building it first if its sources changed) and declare signatures."""
    global _LIB
    with _LIB_LOCK:
        if _LIB is not None and path is None:
            return _LIB
        lib_path = Path(path) if path is not None else _build.build()
        lib = ctypes.CDLL(str(lib_path))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        if path is None:
            _LIB = lib
        return lib


def last_error(lib: ctypes.CDLL | None = None) -> str:
    raw = (lib or library()).mgc_cuda_last_error()
    return raw.decode() if raw else ""


def check(status: int, what: str, lib: ctypes.CDLL | None = None) -> None:
    """Raise the reference's exception types for a non-zero ABI status."""
    if status == 0:
        return
    msg = last_error(lib)
    if status == 1:
        raise GraphError(msg or "compiled model reported an out-of-range Gather index")
    raise CodegenError(f"{what} failed with status {status}: {msg}")
