"""ctypes binding of ``libb200nn.so`` (declared in include/b200nn.h).

The library is the only compute path: if it cannot be loaded the runtime raises,
there is no fallback.  ``load()`` declares argument types for every entry point so
that a wrong call fails in Python rather than in the kernel.
"""

from __future__ import annotations

import ctypes as C
import os
from pathlib import Path

LIB_NAME = "libb200nn.so"
MAX_DIMS = 6
EW_MAX_INPUTS = 4
EW_MAX_OPS = 12

DTYPE_CODES = {"float32": 0, "float16": 1, "bfloat16": 2, "int32": 3, "int64": 4, "uint8": 5, "bool": 5}
DTYPE_BYTES = {"float32": 4, "float16": 2, "bfloat16": 2, "int32": 4, "int64": 8, "uint8": 1, "bool": 1}

EPI_RELU = 1
EPI_SILU_MUL = 2
EPI_GLU = 4
EPI_W_STATIC = 8

MASK_TILE = 128   # rows and keys of a tile of b200_mask_tiles
STEM_TMA_WIDTH = 240   # widest image that b200_conv_stem_pool brings in by TMA (rows of whole 16-byte words)


class Tensor(C.Structure):
    """``b200_tensor``."""

    _fields_ = [("data", C.c_void_p), ("dtype", C.c_int32), ("ndim", C.c_int32),
                ("shape", C.c_int64 * MAX_DIMS), ("stride", C.c_int64 * MAX_DIMS)]


class EwOp(C.Structure):
    """``b200_ew_op``."""

    _fields_ = [("opcode", C.c_int32), ("a", C.c_int32), ("b", C.c_int32), ("round_dtype", C.c_int32), ("imm", C.c_float)]


class PagedAppendArgs(C.Structure):
    """``b200_paged_append_args``."""

    _fields_ = [(n, C.c_void_p) for n in ("q", "k", "v", "cos_t", "sin_t", "q_out", "k_pages", "v_pages", "slots")] + \
               [("n_tokens", C.c_int64), ("num_pages", C.c_int64), ("q_strides", C.c_int64 * 2), ("k_strides", C.c_int64 * 2), ("v_strides", C.c_int64 * 2),
                ("kv_strides", C.c_int64 * 3)] + [(n, C.c_int32) for n in ("Hq", "Hkv", "D", "page_size", "table_dtype", "dtype")]


class AttnPagedArgs(C.Structure):
    """``b200_attn_paged_args``."""

    _fields_ = [(n, C.c_void_p) for n in ("q", "k_pages", "v_pages", "out", "q_start", "kv_len", "page_table", "workspace")] + \
               [(n, C.c_int64) for n in ("workspace_bytes", "B", "n_tokens", "max_q", "num_pages", "table_stride")] + \
               [("q_strides", C.c_int64 * 2), ("kv_strides", C.c_int64 * 3), ("window", C.c_int64)] + \
               [(n, C.c_int32) for n in ("Hq", "Hkv", "D", "page_size", "dtype")] + [("scale", C.c_float)]


_vp, _i, _i64, _f = C.c_void_p, C.c_int, C.c_int64, C.c_float
_TP = C.POINTER(Tensor)
_I64P = C.POINTER(C.c_int64)

# name -> (restype, argtypes); every symbol include/b200nn.h declares
SIGNATURES = {
    "b200_version": (_i, []),
    "b200_last_error": (C.c_char_p, []),
    "b200_device_info": (_i, [_i, C.POINTER(_i), C.POINTER(_i), C.POINTER(_i), C.POINTER(_i64)]),
    "b200_debug_device_error": (_i, [C.POINTER(_i), _i]),
    "b200_debug_wait_timeout": (_i, [_i, _vp]),
    "b200_ew_chain": (_i, [_TP, _TP, _i, C.POINTER(EwOp), _i, _vp]),
    "b200_strided_copy": (_i, [_TP, _TP, _vp]),
    "b200_fill": (_i, [_vp, _i64, C.c_double, _i, _vp]),
    "b200_rmsnorm": (_i, [_vp, _vp, _vp, _i64, _i64, _i64, _i64, _f, _i, _i, _vp]),
    "b200_softmax": (_i, [_vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _f, _i, _i, _i, _i, _vp]),
    "b200_mean_last_dim": (_i, [_vp, _vp, _i64, _i64, _i, _i, _vp]),
    "b200_embedding": (_i, [_vp, _vp, _vp, _i64, _i64, _i64, _i, _vp]),
    "b200_index_copy": (_i, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i, _i, _vp]),
    "b200_argmax_rows": (_i, [_vp, _vp, _i64, _i64, _i64, _i, _vp]),
    "b200_rope_table": (_i, [_vp, _vp, _vp, _vp, _i64, _i, _i, _i, _vp]),
    "b200_rope_rotate": (_i, [_TP, _vp, _vp, _vp, _vp, _vp, _i64, _i, _vp]),
    "b200_rope_rotate_pair": (_i, [_TP, _TP, _vp, _vp, _vp, _vp, _vp]),
    "b200_qkv_rope_cache": (_i, [_TP, _TP, _TP, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i, _vp]),
    "b200_max_pool2d": (_i, [_TP, _TP, _i, _i, _i, _i, _i, _i, _vp]),
    "b200_adaptive_avg_pool2d": (_i, [_TP, _TP, _vp]),
    "b200_batch_norm": (_i, [_TP, _TP, _vp, _vp, _vp, _vp, _f, _i, _i, _vp]),
    "b200_conv_weight_prep": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _f, _i, _i, _i, _vp]),
    "b200_linear": (_i, [_vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i, _i, _i, _vp, _i64, _vp, _i64, _vp]),
    "b200_linear_workspace_bytes": (_i64, [_i64, _i64, _i64]),
    "b200_linear_rmsnorm": (_i, [_vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i, _i, _i, _vp, _i64, _vp, _vp, _i64, _f, _i, _vp]),
    "b200_linear_norm": (_i, [_vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i, _i, _i, _f, _vp, _i, _vp, _vp]),
    "b200_linear_qkv_rope": (_i, [_vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i, _i, _i, _f, _vp, _i, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i, _i, _i,
                                  _vp]),
    "b200_matmul_strided": (_i, [_vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _I64P, _I64P, _I64P, _i, _vp]),
    "b200_conv2d_nhwc": (_i, [_vp, _vp, _vp, _vp, _vp] + [_i] * 16 + [_vp]),
    "b200_conv_stem_pool": (_i, [_vp, _vp, _vp, _vp] + [_i] * 14 + [_vp]),
    "b200_conv_stem_pool_supported": (_i, [_i] * 12),
    "b200_attn_decode": (_i, [_vp, _vp, _vp, _vp, _vp, _i64, _i, _i, _i64, _i, _i64, _i64, _i64, _i64, _f, _i, _vp, _i64, _vp]),
    "b200_attn_decode_noalloc": (_i, [_vp, _vp, _vp, _vp, _vp, _i64, _i, _i, _i64, _i, _i64, _i64, _i64, _i64, _f, _i, _vp]),
    "b200_attn_decode_workspace_bytes": (_i64, [_i64, _i, _i, _i64, _i]),
    "b200_attn_prefill_tiles": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _i64, _i, _i, _i64, _i64, _i, _I64P, _I64P, _I64P, _i64, _i64, _f, _i, _vp]),
    "b200_attn_prefill_reads_tiles": (_i, [_vp, _i64, _i64, _i64, _i]),
    "b200_mask_tiles": (_i, [_vp, _i64, _i64, _i64, _i64, _i64, _i, _vp, _vp]),
    "b200_attn_prefill": (_i, [_vp, _vp, _vp, _vp, _vp, _i64, _i, _i, _i64, _i64, _i, _I64P, _I64P, _I64P, _i64, _i64, _f, _i, _vp]),
    "b200_paged_append": (_i, [_vp, _vp]),   # PagedAppendArgs, stream
    "b200_attn_paged": (_i, [_vp, _vp]),     # AttnPagedArgs, stream
    "b200_attn_paged_workspace_bytes": (_i64, [_i64, _i, _i, _i]),
    "b200_sample_rows": (_i, [_vp, _vp, _i64, _i64, _i64, _vp, _vp, _vp, _vp, _vp, _i, _vp]),
}

_lib = None
_test_override = None  # (library object, torch device string) installed by the test-suite


def library_path() -> Path:
    env = os.environ.get("B200NN_LIBRARY")
    return Path(env) if env else Path(__file__).resolve().parent / LIB_NAME


def load():
    """The loaded library with typed entry points.  Raises ``RuntimeError`` when the
    shared object is missing or does not export a declared symbol."""
    global _lib
    if _test_override is not None:
        return _test_override[0]
    if _lib is not None:
        return _lib
    path = library_path()
    if not path.exists():
        raise RuntimeError(f"{path} not found: build it with `python build_native.py` (needs nvcc); "
                           "there is no fallback path without the native kernel library")
    try:
        lib = C.CDLL(str(path))
    except OSError as exc:
        raise RuntimeError(f"cannot load {path}: {exc}") from exc
    for name, (restype, argtypes) in SIGNATURES.items():
        try:
            fn = getattr(lib, name)
        except AttributeError as exc:
            raise RuntimeError(f"{path} does not export {name}") from exc
        fn.restype = restype
        fn.argtypes = argtypes
    _lib = lib
    return lib


def device_string(device_id: int = 0) -> str:
    if _test_override is not None:
        return _test_override[1]
    return f"cuda:{device_id}"


def install_test_library(lib, device: str = "cpu") -> None:
    """Test seam: route calls to a stand-in object (used by the CPU test-suite to
    exercise the host logic without a GPU).  Never used by the product."""
    global _test_override
    _test_override = None if lib is None else (lib, device)


_calls = None
_entries: dict = {}   # name -> (library, address, what must stay alive for it)


def torch_calls_built_for() -> str:
    """What a ``b200_torch_calls`` that can be loaded into this process carries in it (its code depends on the layout of torch's classes)."""
    import sys

    import torch

    return f"b200_torch_calls for torch {torch.__version__}, {sys.implementation.cache_tag}"


def torch_calls():
    """The module ``b200_torch_calls`` (csrc/torch_calls.cpp): entry points called with torch tensors."""
    global _calls
    if _calls is None:
        import importlib.machinery
        import importlib.util

        import torch  # noqa: F401  (its libraries first)

        path = Path(__file__).resolve().parent / "b200_torch_calls.so"
        if not path.exists():
            raise RuntimeError(f"{path} not found: build it with `python build_native.py`; there is no fallback path without it")
        if torch_calls_built_for().encode() not in path.read_bytes():
            raise RuntimeError(f"{path} was built for another torch than {torch.__version__}: build it again with `python build_native.py`")
        loader = importlib.machinery.ExtensionFileLoader("b200_torch_calls", str(path))
        _calls = importlib.util.module_from_spec(importlib.util.spec_from_loader("b200_torch_calls", loader))
        loader.exec_module(_calls)
    return _calls


def entry(name: str) -> int:
    """Entry point ``name`` for ``torch_calls``: its address in the library, which takes CUDA tensors, or minus that of the test stand-in's."""
    lib = _test_override[0] if _test_override is not None else _lib or load()
    got = _entries.get(name)
    if got is None or got[0] is not lib:
        fn = getattr(lib, name)
        stand_in = not isinstance(lib, C.CDLL)
        if stand_in:
            restype, argtypes = SIGNATURES[name]
            fn = C.CFUNCTYPE(restype, *argtypes)(fn)
        address = C.cast(fn, C.c_void_p).value
        got = _entries[name] = (lib, -address if stand_in else address, fn)
    return got[1]


def check(rc: int, what: str = "") -> None:
    if rc != 0:
        msg = load().b200_last_error()
        msg = msg.decode() if isinstance(msg, bytes) else str(msg)
        raise RuntimeError(f"b200nn call failed ({rc}) {what}: {msg}")


def make_tensor(ptr: int, dtype: str, shape, strides) -> Tensor:
    if len(shape) > MAX_DIMS:
        raise ValueError(f"tensor rank {len(shape)} exceeds {MAX_DIMS}")
    t = Tensor()
    t.data = ptr
    t.dtype = DTYPE_CODES[dtype]
    t.ndim = len(shape)
    for i, (s, st) in enumerate(zip(shape, strides)):
        t.shape[i] = int(s)
        t.stride[i] = int(st)
    return t
