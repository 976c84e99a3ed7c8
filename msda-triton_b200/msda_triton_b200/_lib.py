"""ctypes binding of ``libmsda_b200.so`` (C ABI declared in include/msda_b200.h
and include/msda_layer_b200.h).

The library is loaded lazily on first use. If it is missing or cannot be
loaded the op raises ``RuntimeError``: there is no fallback implementation.
"""

from __future__ import annotations

import ctypes
import os
import threading
from pathlib import Path

LIB_PATH = Path(os.environ.get("MSDA_B200_LIB") or (Path(__file__).resolve().parent / "libmsda_b200.so"))

MSDA_OK = 0
MSDA_ERR_INVALID_ARGUMENT = 1
MSDA_ERR_UNSUPPORTED = 2
MSDA_ERR_CUDA = 3

MSDA_DTYPE_F32 = 0
MSDA_DTYPE_F16 = 1
MSDA_DTYPE_BF16 = 2

MSDA_BWD_FP32_ACCUM = 1
MSDA_BWD_FORCE_SCATTER = 2
MSDA_BWD_FORCE_COUNTED = 8
MSDA_BWD_DETERMINISTIC = 16
MSDA_BWD_GRAD_INPUT_NCHW = 32

MSDA_POSITION_F32 = 0
MSDA_POSITION_I32 = 1
MSDA_POSITION_I64 = 2
MSDA_ROTARY_MAX_AXES = 8
MSDA_ROTARY_MAX_HEAD_DIM = 512
MSDA_LAYER_NORM_MAX_WIDTH = 1 << 20
MSDA_ATTENTION_MAX_HEAD_DIM = 256

# Every symbol include/msda_b200.h and include/msda_layer_b200.h declare, with
# (restype, argtypes).
_VP = ctypes.c_void_p
_I64 = ctypes.c_int64
_I32 = ctypes.c_int32
SIGNATURES = {
    "msda_version": (ctypes.c_char_p, []),
    "msda_last_error": (ctypes.c_char_p, []),
    "msda_forward": (
        ctypes.c_int,
        [_VP, _VP, _VP, _VP, _VP, _VP, _I64, _I64, _I64, _I32, _I32, _I32, _I32, _I32, _VP],
    ),
    "msda_backward_workspace_size": (
        ctypes.c_size_t, [_I64, _I64, _I64, _I32, _I32, _I32, _I32, _I32, ctypes.c_uint32]),
    "msda_backward": (
        ctypes.c_int,
        [_VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, ctypes.c_size_t,
         _I64, _I64, _I64, _I32, _I32, _I32, _I32, _I32, ctypes.c_uint32, _VP],
    ),
    # Fused layer prologue: reference points + offsets (level pixels) and
    # attention logits instead of locations and weights.
    "msda_forward_fused": (
        ctypes.c_int,
        [_VP, _VP, _VP, _VP, _VP, _VP, _VP, _I64, _I64, _I64, _I32, _I32, _I32, _I32, _I32, _VP],
    ),
    "msda_backward_fused": (
        ctypes.c_int,
        [_VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, ctypes.c_size_t,
         _I64, _I64, _I64, _I32, _I32, _I32, _I32, _I32, ctypes.c_uint32, _VP],
    ),
    # The backward for callers that cannot allocate: same as msda_backward
    # without the workspace arguments (fp32 scratch from a static device array).
    "msda_backward_noalloc": (
        ctypes.c_int,
        [_VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP,
         _I64, _I64, _I64, _I32, _I32, _I32, _I32, _I32, _VP],
    ),
    # Sibling gathers on NHWC data: grid_sample and ROI-Align; the layout conversion.
    "msda_transpose": (ctypes.c_int, [_VP, _VP, _I64, _I64, _I64, _I32, _VP]),
    "msda_grid_sample_forward": (
        ctypes.c_int, [_VP, _VP, _VP, _I64, _I64, _I64, _I64, _I64, _I64, _I32, _I32, _I32, _I32, _VP]),
    "msda_grid_sample_backward_workspace_size": (
        ctypes.c_size_t, [_I64, _I64, _I64, _I64, _I64, _I64, _I32, ctypes.c_uint32]),
    "msda_grid_sample_backward": (
        ctypes.c_int,
        [_VP, _VP, _VP, _VP, _VP, _VP, ctypes.c_size_t, _I64, _I64, _I64, _I64, _I64, _I64,
         _I32, _I32, _I32, _I32, ctypes.c_uint32, _VP],
    ),
    "msda_roi_align_forward": (
        ctypes.c_int,
        [_VP, _VP, _VP, _I64, _I64, _I64, _I64, _I64, _I32, _I32, ctypes.c_float, _I32, _I32,
         _I32, _VP],
    ),
    "msda_roi_align_backward_workspace_size": (
        ctypes.c_size_t, [_I64, _I64, _I64, _I64, _I32, ctypes.c_uint32]),
    "msda_roi_align_backward": (
        ctypes.c_int,
        [_VP, _VP, _VP, _VP, ctypes.c_size_t, _I64, _I64, _I64, _I64, _I64, _I32, _I32,
         ctypes.c_float, _I32, _I32, _I32, ctypes.c_uint32, _VP],
    ),
    # include/msda_layer_b200.h: the operators beside the sampling.
    "msda_rotary": (
        ctypes.c_int,
        [_VP, _VP, _VP, _VP, _VP, _I64, _I64, _I32, _I32, _I32, _VP, _VP, _I64, _I32, _I32, _VP,
         ctypes.c_double, _I32, _I32, _I32, _I32, _VP],
    ),
    "msda_layer_norm_forward": (
        ctypes.c_int,
        [_VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _I64, _I64, _I64, _I64, ctypes.c_float, _I32, _I32, _VP],
    ),
    "msda_layer_norm_backward_workspace_size": (ctypes.c_size_t, [_I64, _I64]),
    "msda_layer_norm_backward": (
        ctypes.c_int,
        [_VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, ctypes.c_size_t,
         _I64, _I64, _I64, _I64, _I64, _I32, _I32, _VP],
    ),
    "msda_attention_workspace_size": (ctypes.c_size_t, [_VP, _I32]),
    "msda_attention_forward": (ctypes.c_int, [_VP, _VP]),
    "msda_attention_backward": (ctypes.c_int, [_VP, _VP]),
    "msda_attention_gave_up": (ctypes.c_int, [ctypes.POINTER(_I32)]),
}

# Size of the static scratch behind msda_backward_noalloc
# (MSDA_NOALLOC_SCRATCH_BYTES in include/msda_b200.h).
MSDA_NOALLOC_SCRATCH_BYTES = 16 << 20


class AttentionArgs(ctypes.Structure):
    """msda_attention_args of include/msda_layer_b200.h."""

    _fields_ = [
        (n, ctypes.c_void_p) for n in ("query", "key", "value", "out", "out_residue", "lse", "grad_out", "grad_query", "grad_key",
                                       "grad_value")
    ] + [
        (n, ctypes.c_int64) for n in ("batch", "num_queries", "num_keys")
    ] + [
        (n, ctypes.c_int32) for n in ("num_heads", "num_key_heads", "head_dim", "dtype")
    ] + [
        (n, ctypes.c_int64 * 3) for n in ("query_strides", "key_strides", "value_strides", "grad_out_strides")
    ] + [
        ("scale", ctypes.c_float), ("softcap", ctypes.c_float)
    ] + [
        (n, ctypes.c_void_p) for n in ("distance_slopes", "query_documents", "key_documents", "prefix_lengths",
                                       "key_lengths")
    ] + [
        ("shared_document", ctypes.c_int32), ("causal", ctypes.c_int32),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
    ]


_lock = threading.Lock()
_lib: ctypes.CDLL | None = None


class MSDALibraryError(RuntimeError):
    """A call into libmsda_b200 returned a non-zero status."""

    def __init__(self, fn: str, code: int, message: str):
        super().__init__(f"{fn} failed with status {code}: {message}")
        self.code = code


def load() -> ctypes.CDLL:
    """Load the shared library (once) and declare its signatures."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"the msda_b200 CUDA library is not built ({LIB_PATH} is missing); "
                "run `python -m msda_triton_b200.build` or __graft_entry__.build()"
            )
        try:
            lib = ctypes.CDLL(str(LIB_PATH))
        except OSError as exc:  # pragma: no cover - depends on the host
            raise RuntimeError(f"cannot load {LIB_PATH}: {exc}") from exc
        for name, (restype, argtypes) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = restype
            fn.argtypes = argtypes
        _lib = lib
        return lib


def check(fn_name: str, code: int) -> None:
    if code != MSDA_OK:
        msg = load().msda_last_error().decode(errors="replace")
        raise MSDALibraryError(fn_name, code, msg)


def version() -> str:
    return load().msda_version().decode()
