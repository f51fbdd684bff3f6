"""
ctypes binding of libbgmm_ops.so (the C-ABI of include/bgmm_ops.h) for torch tensors.

There is NO CPU fallback: tensors that are not on a HIP device are refused.
"""
import ctypes
import os

import torch

from .. import _build
from .._lib import BGMMError

_vp, _i32, _i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64

LEVELS = 12                 # tile sizes of a grouping (include/bgmm_ops.h: BGMM_OPS_LEVELS)
MAX_COMPONENTS = 8000
MAX_CHOSEN = 32

DTYPES = {torch.float64: 0, torch.float32: 1, torch.float16: 2, torch.bfloat16: 3}

# every symbol include/bgmm_ops.h declares: name -> (restype, argtypes)
SIGNATURES = {
    "bgmm_ops_last_error": (ctypes.c_char_p, []),
    "bgmm_ops_runtime_path": (ctypes.c_char_p, []),
    "bgmm_group_rows_ws": (_i64, [_i64, _i32]),
    "bgmm_group_rows_tiles": (_i64, [_i64, _i32]),
    "bgmm_group_rows": (_i32, [_vp, _i64, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _vp]),
    "bgmm_rows_product_splits": (_i32, [_i32, _i64, _i32, _i32, _i32]),
    "bgmm_rows_product": (_i32, [_i32, _vp, _i64, _i32, _vp, _i64, _i64, _i32, _vp, _i64, _vp, _vp, _i64, _vp, _i32, _i64, _i32, _i32, _i32,
                                 _vp, _vp, _vp]),
    "bgmm_weight_product_ws": (_i64, [_i32, _i64, _i32, _i32, _i32]),
    "bgmm_weight_product": (_i32, [_i32, _vp, _i64, _i32, _vp, _i64, _i32, _vp, _vp, _vp, _vp, _i64, _i64, _i32, _i32, _i32, _vp, _vp, _vp, _vp]),
    "bgmm_combine": (_i32, [_i32, _vp, _i32, _i64, _i32, _i32, _vp, _vp, _vp, _i64, _i32, _vp, _vp, _i64, _vp, _i64, _vp, _i64, _i32, _i32, _vp]),
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
        _build.build()
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


def check(rc):
    if rc != 0:
        raise BGMMError(rc, (_lib.bgmm_ops_last_error() or b"").decode())


def refuse(message, *args, code=-1):
    """An argument that an operator does not take: BGMM_EINVAL (or the code given), as the library's own."""
    raise BGMMError(code, message % args)


def require_tensors(what, **tensors):
    for name, t in tensors.items():
        if t is not None and not isinstance(t, torch.Tensor):
            refuse("%s: %s is no torch tensor", what, name)


def require_device(what, **tensors):
    """All the tensors given (None: absent) on one HIP device; returns it."""
    device = None
    for name, t in tensors.items():
        if t is None:
            continue
        d = t.device
        if d.type != "cuda":
            refuse("%s: %s is on %s; the operators run on HIP devices only", what, name, d, code=-2)
        if device is None:
            device = d
        elif d != device:
            refuse("%s: %s is on %s, the others on %s", what, name, d, device)
    return device


class _Here(object):
    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_here = _Here()


def on(device):
    """Context with `device` current (nothing to do, and nothing paid, where it is already)."""
    return _here if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def acc_dtype(dtype):
    """What products and sums of an element type are held in."""
    return torch.float64 if dtype == torch.float64 else torch.float32


def ptr(t):
    return None if t is None else t.data_ptr()


def stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)
