"""ctypes binding of the C ABI in ``include/llm_kernels_b200.h`` (``liblk_b200.so``).

The Python layer reaches the GPU only through these entry points, with raw device pointers,
element strides and torch's current CUDA stream: by ctypes, or for the serving operators, whose
calls are small, by a CPython extension over the same library (``binding``).  There is no other
code path — if the library is missing, the ops raise instead of computing anything.
"""

from __future__ import annotations

import ctypes
import os
import threading

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "liblk_b200.so")

# Status codes (lk_status) and dtype codes (lk_dtype) of the header.
LK_OK = 0
LK_ERR_INVALID_ARG = 1
LK_ERR_UNSUPPORTED = 2
LK_ERR_CUDA = 3
LK_ERR_TIMEOUT = 4
LK_ERR_ALIGNMENT = 5
LK_ERR_SCRATCH_LIMIT = 6
LK_PEER_HANDLE_BYTES = 64  # include/llm_kernels_b200.h

LK_F32, LK_F16, LK_BF16, LK_I8, LK_I32, LK_I64 = 0, 1, 2, 3, 4, 5

# Failure-path test hooks (lk_inject).
LK_INJECT_NONE, LK_INJECT_FA_DROP_LOAD, LK_INJECT_GEMM_DROP_LOAD, LK_INJECT_SPLIT_SKIP_PUBLISH = 0, 1, 2, 3
LK_INJECT_REQUANT_SKIP_PUBLISH, LK_INJECT_PAGED_DROP_LOAD = 4, 5

_p = ctypes.c_void_p
_i = ctypes.c_int
_i64 = ctypes.c_int64
_f = ctypes.c_float
_pi64 = ctypes.POINTER(ctypes.c_int64)

# name -> (restype, argtypes); mirrors include/llm_kernels_b200.h one for one.
SIGNATURES = {
    "lk_status_string": (ctypes.c_char_p, [_i]),
    "lk_last_cuda_error": (_i, []),
    "lk_version": (_i, []),
    "lk_set_device": (_i, [_i]),
    "lk_device_status": (_i, [ctypes.POINTER(ctypes.c_int)]),
    "lk_clear_device_status": (_i, []),
    "lk_debug_set_wait_limit": (_i, [_i64]),
    "lk_debug_inject": (_i, [_i, _i, _i]),
    "lk_quantize_symmetric": (_i, [_p, _i, _i64, _i64, _i64, _p, _i64, _p, _p]),
    "lk_int8_gemm_dequant": (_i, [_p, _i64, _p, _i64, _i, _p, _p, _p, _i64, _i64, _i64, _i64, _p]),
    "lk_int8_gemm_i32": (_i, [_p, _i64, _p, _i64, _i, _p, _i64, _i64, _i64, _i64, _p]),
    "lk_int8_gemm_requant_workspace_bytes": (_i64, [_i64]),
    "lk_int8_gemm_dequant_requant": (
        _i, [_p, _i64, _p, _i64, _i, _p, _p, _p, _i64, _p, _i64, _p, _p, _i64, _i64, _i64, _p],
    ),
    "lk_int8_gemm_dequant_scatter": (
        _i, [_p, _i64, _p, _i64, _i, _p, _p, _p, _i, _i64, _i64, _i64, _i64, _i64, _p],
    ),
    "lk_int8_gemm_dequant_multicast": (
        _i, [_p, _i64, _p, _i64, _i, _p, _p, _p, _i64, _i64, _i64, _i64, _i64, _p],
    ),
    "lk_peer_export": (_i, [_i, _p, _p, _pi64]),
    "lk_peer_open": (_i, [_i, _p, _i64, ctypes.POINTER(ctypes.c_void_p)]),
    "lk_peer_close": (_i, [_i, _p, _i64]),
    "lk_flash_attn_fwd": (
        _i,
        [_p, _p, _p, _p, _i, _i64, _i64, _i64, _i64, _i64, _pi64, _pi64, _pi64, _pi64, _i, _f, _p],
    ),
    "lk_flash_attn_fwd_gqa": (
        _i,
        [_p, _p, _p, _p, _i, _i64, _i64, _i64, _i64, _i64, _i64, _pi64, _pi64, _pi64, _pi64, _i, _f, _p],
    ),
    "lk_flash_attn_fwd_lse": (
        _i,
        [_p, _p, _p, _p, _p, _i64, _i, _i64, _i64, _i64, _i64, _i64, _i64, _pi64, _pi64, _pi64, _pi64, _i, _f, _p],
    ),
    "lk_flash_attn_bwd": (
        _i,
        [_p, _p, _p, _p, _p, _p, _i64, _p, _p, _p, _p, _i, _i64, _i64, _i64, _i64, _i64, _i64, _pi64, _i, _f, _p],
    ),
    "lk_rotary_embed": (
        _i,
        [_p, _p, _p, _p, _pi64, _i, _i64, _i64, _i64, _i64, _i64, _p, _i, _pi64, _p, _i64, _i64, _i64, _pi64, _i, _i, _p],
    ),
    "lk_paged_kv_append": (
        _i,
        [_p, _p, _p, _p, _p, _p, _pi64, _i, _i64, _i64, _i64, _i64, _i64, _i64, _p, _i, _p, _i, _pi64, _p, _i64, _i64,
         _i64, _pi64, _i, _p],
    ),
    "lk_paged_attention_workspace_bytes": (_i64, [_i64, _i64, _i64, _i64, _i64, _i64]),
    "lk_paged_attention": (
        _i,
        [_p, _p, _p, _p, _i64, _i64, _p, _p, _p, _pi64, _i, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _f, _p, _i64, _p],
    ),
    "lk_shared_prefix_attention": (
        _i,
        [_p, _p, _p, _p, _i64, _p, _i64, _i64, _p, _p, _p, _pi64, _i, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _f, _p,
         _i64, _p],
    ),
    "lk_rmsnorm_linear_fold": (_i, [_p, _i, _p, _p, _i, _i64, _i64, _p]),
    "lk_rmsnorm_linear": (_i, [_p, _i64, _p, _p, _i64, _i, _i64, _i64, _i64, _f, _p, _p]),
    "lk_fused_rmsnorm_linear": (_i, [_p, _p, _p, _p, _f, _i64, _i64, _i64, _i, _p, _p, _p]),
    "lk_rmsnorm_linear_noalloc": (_i, [_p, _i64, _p, _p, _i64, _i, _i64, _i64, _i64, _f, _p]),
}

_lib = None
_lock = threading.Lock()


class LKError(RuntimeError):
    """A C-ABI call returned a failure status."""

    def __init__(self, fn: str, status: int, detail: str = ""):
        self.status = status
        msg = f"{fn}: {status_string(status)} (status {status})"
        if detail:
            msg += f": {detail}"
        super().__init__(msg)


def load() -> ctypes.CDLL:
    """Loads ``liblk_b200.so`` (once) and declares every entry point's signature."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not os.path.exists(LIB_PATH):
            raise ImportError(
                f"llm_kernels: native library {LIB_PATH} is missing; build it with "
                "`python flash-attn-from-scratch_b200/build.py` (nvcc, sm_100a)"
            )
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


_binding = None


def _capturing(device: int) -> bool:
    """Whether torch's current stream on ``device``, which need not be the current one, is being captured."""
    import torch

    if device == torch.cuda.current_device():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def _call_error(name: str, status: int, cuda: int) -> LKError:
    return LKError(name, status, f"cudaError {cuda}" if cuda else "")


def binding():
    """The CPython extension of the serving operators (csrc/binding.cpp), set up once."""
    global _binding
    if _binding is not None:
        return _binding
    load()
    with _lock:
        if _binding is None:
            import torch

            from ._common import LKInputError

            try:
                from . import _binding as ext
            except ImportError as e:
                raise ImportError(
                    "llm_kernels: the extension of the serving operators (llm_kernels/_binding.so) is missing; build it with "
                    "`python flash-attn-from-scratch_b200/build.py` where g++ and the headers of Python and torch are"
                ) from e

            ext.setup(
                torch.Tensor,
                torch.empty_like,
                lambda q: torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device),
                _capturing,
                lambda dev, n: torch.zeros(n, dtype=torch.uint8, device=torch.device("cuda", dev)),
                LKInputError,
                _call_error,
            )
            _binding = ext
    return _binding


def status_string(status: int) -> str:
    try:
        return load().lk_status_string(int(status)).decode()
    except Exception:  # pragma: no cover - only when the library itself failed to load
        return "unknown"


def call(name: str, *args) -> None:
    """Calls entry point ``name`` and raises LKError on a non-zero status."""
    lib = load()
    st = getattr(lib, name)(*args)
    if st != LK_OK:
        detail = ""
        if st == LK_ERR_CUDA:
            detail = f"cudaError {lib.lk_last_cuda_error()}"
        raise LKError(name, st, detail)


def i64_array(vals) -> ctypes.Array:
    return (ctypes.c_int64 * len(vals))(*[int(v) for v in vals])


def set_device(index: int) -> None:
    """Picks the device of this thread's calls on the default stream; torch's current device stays."""
    if (_lib or load()).lk_set_device(index) != LK_OK:  # on the way of every call
        call("lk_set_device", index)


def device_status() -> tuple[int, int, int, int]:
    """Synchronises and returns the device status word (code, site, block, thread): code 4 for a
    pipeline wait that ran out, 1 for an index out of range in device data (a cache slot, a page
    id, a position, a length).  The device is that of this thread's last call, or torch's current
    one if that has been changed since."""
    out = (ctypes.c_int * 4)()
    st = load().lk_device_status(out)
    if st not in (LK_OK, LK_ERR_TIMEOUT, LK_ERR_INVALID_ARG):
        raise LKError("lk_device_status", st)
    return tuple(out)


def clear_device_status() -> None:
    call("lk_clear_device_status")
    if _binding is not None:
        _binding.drop_workspaces()  # their counters are not to be trusted after a failure


def exported_symbols() -> list[str]:
    return list(SIGNATURES)
