"""
Loading of libbgmm_ops.so (the C-ABI of include/bgmm_ops.h) and of its torch binding.

There is NO CPU fallback: tensors that are not on a HIP device are refused, and a library that is missing and cannot be
built raises.
"""
import ctypes
import os

import torch

from .. import _build

_vp, _i32, _i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64

LEVELS = 8                  # chunk sizes of a grouping (include/bgmm_ops.h: BGMM_OPS_LEVELS)
MAX_COMPONENTS = 8000
MAX_CHOSEN = 32

# every symbol include/bgmm_ops.h declares: name -> (restype, argtypes)
SIGNATURES = {
    "bgmm_ops_last_error": (ctypes.c_char_p, []),
    "bgmm_ops_runtime_path": (ctypes.c_char_p, []),
    "bgmm_group_rows_ws": (_i64, [_i64, _i32]),
    "bgmm_group_rows_tiles": (_i64, [_i64, _i32]),
    "bgmm_group_rows": (_i32, [_vp, _i64, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _vp]),
    "bgmm_rows_product_splits": (_i32, [_i32, _i64, _i32, _i32, _i32]),
    "bgmm_rows_product_dots": (_i32, [_i32, _i64, _i32, _i32, _i32, _i32]),
    "bgmm_rows_product": (_i32, [_i32, _vp, _i64, _i32, _vp, _i64, _i64, _i32, _vp, _i64, _vp, _vp, _i64, _vp, _i32, _vp, _i64, _i32, _vp,
                                 _i64, _i32, _i32, _i32, _vp, _vp, _vp]),
    "bgmm_weight_product_ws": (_i64, [_i32, _i64, _i32, _i32, _i32]),
    "bgmm_weight_product": (_i32, [_i32, _vp, _i64, _i32, _vp, _i64, _i32, _vp, _vp, _vp, _vp, _i64, _i64, _i32, _i32, _i32, _vp, _vp, _vp, _vp]),
    "bgmm_combine": (_i32, [_i32, _vp, _i32, _i64, _i32, _i32, _vp, _vp, _vp, _i64, _i32, _vp, _vp, _i64, _vp, _i64, _vp, _i64, _i32, _i32, _vp]),
    "bgmm_gate_gradient": (_i32, [_i32, _vp, _i32, _i64, _i32, _vp, _vp, _i64, _vp, _i64, _i32, _i32, _vp, _vp]),
    "bgmm_route": (_i32, [_i32, _vp, _i64, _i64, _i32, _i32, _i32, _vp, _vp, _vp, _vp]),
    "bgmm_route_backward": (_i32, [_i32, _vp, _i64, _i64, _i32, _i32, _i32, _vp, _vp, _vp, _vp, _vp, _vp]),
    "bgmm_verify_drafts": (_i32, [_i32, _vp, _i64, _i64, _vp, _i64, _i64, _vp, _vp, _vp, _vp, _i64, _i32, _i64, _vp, _vp, _vp, _i64, _vp]),
    "bgmm_verify_drafts_ws": (_i64, [_i64, _i64]),
}

_lib = None


def load():
    """Load the library (building it first if it is absent), bound to the HIP runtime that torch uses."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(_build.OPS_LIB):
        _build.build_ops()
    # The library links no HIP runtime.  libbgmm_hip.so may have brought the system's into the process; streams and device
    # pointers of one runtime mean nothing to the other, so torch's copy is made visible first and the binding is checked.
    runtime = os.path.join(os.path.dirname(torch.__file__), "lib", "libamdhip64.so")
    ctypes.CDLL(runtime, mode=ctypes.RTLD_GLOBAL)
    L = ctypes.CDLL(_build.OPS_LIB)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    bound = L.bgmm_ops_runtime_path().decode()
    if not (os.path.exists(bound) and os.path.samefile(bound, runtime)):
        raise OSError("libbgmm_ops.so is bound to %s, but torch runs on %s" % (bound, runtime))
    _lib = L
    return L


def binding():
    """The extension module with the operators (csrc/ops_torch.cpp)."""
    if not os.path.exists(_build.OPS_BINDING):
        _build.build_ops()
    load()                              # (first: it settles which HIP runtime the library binds to)
    from . import _binding
    return _binding
