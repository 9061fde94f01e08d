"""ctypes binding of the int8 operators' C ABI (``include/w4a8_int8.h``, ``libw4a8int8.so``).

Loading fails loudly: there is no CPU or Python fallback for any kernel.
"""
from __future__ import annotations

import ctypes
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libw4a8int8.so"

_p = ctypes.c_void_p
_i64 = ctypes.c_int64
_int = ctypes.c_int
_size = ctypes.c_size_t

# name -> (restype, argtypes); must match include/w4a8_int8.h exactly.
SIGNATURES = {
    "w4a8_int8_abi_version": (_int, []),
    "w4a8_int8_last_error": (ctypes.c_char_p, []),
    "w4a8_act_quant_int8": (_int, [_p, _int, _i64, _i64, _i64, _int, _p, _p, _p]),
    "w4a8_int8_gemm_workspace_size": (_size, [_int, _i64, _i64, _i64]),
    "w4a8_int8_gemm": (_int, [_p, _int, _p, _i64, _i64, _i64, _p, _p, _i64, _p, _int, _p, _int, _p, _size, _p]),
    "w4a8_moe_int8_workspace_size": (_size, [_i64, _i64, _i64, _i64, _i64]),
    "w4a8_moe_int8_apply": (_int, [_p, _int, _p, _i64, _i64, _i64, _i64, _i64, _p, _p, _p, _p, _p, _p, _p, _i64, _p,
                                   _int, _p, _size, _p]),
}

ABI_VERSION = 1


def _load() -> ctypes.CDLL:
    if not LIB_PATH.exists():
        raise ImportError(
            f"w4a8_fp8_wmma: HIP library not built ({LIB_PATH}); run "
            "`python rdna4-vllm_amd/build.py` (there is no CPU fallback)")
    lib = ctypes.CDLL(str(LIB_PATH))
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    if lib.w4a8_int8_abi_version() != ABI_VERSION:
        raise ImportError(f"w4a8_fp8_wmma: ABI version mismatch in {LIB_PATH}")
    return lib


lib = _load()


def check(rc: int, what: str) -> None:
    """Raise RuntimeError with the library's message on a non-zero status."""
    if rc != 0:
        msg = (lib.w4a8_int8_last_error() or b"").decode(errors="replace")
        raise RuntimeError(f"{what}: {msg} (status {rc})")
