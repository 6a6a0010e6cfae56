"""ctypes binding of the policy operators' C-ABI (include/urgym_ops.h, liburgym_ops.so), for callers with pointers of their own.

urgym_amd.ops calls the same entries from C++ (urgym_ops_torch.so), with torch's tensors, allocator and streams.
"""
import ctypes
import os

_LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "_lib")
LIB_PATH = os.path.join(_LIB, "liburgym_ops.so")
TORCH_PATH = os.path.join(_LIB, "urgym_ops_torch.so")
# C-ABI symbols declared in include/urgym_ops.h
SYMBOLS = ["urgym_ops_last_error", "urgym_ops_layer_norm", "urgym_ops_layer_norm_workspace", "urgym_ops_layer_norm_backward",
           "urgym_ops_decay_workspace", "urgym_ops_decay_backward_workspace", "urgym_ops_decay",
            "urgym_ops_decay_backward", "urgym_ops_decay_step"]
F32, BF16, F16 = 0, 1, 2
MAX_HEAD_DIM = 128
_lib = None


class Seq(ctypes.Structure):
    """urgym_ops_seq"""
    _fields_ = [("dtype", ctypes.c_int32), ("heads", ctypes.c_int32), ("dk", ctypes.c_int32), ("dv", ctypes.c_int32),
                ("steps", ctypes.c_int64), ("envs", ctypes.c_int64),
                ("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("q_stride", ctypes.c_int64 * 3), ("k_stride", ctypes.c_int64 * 3), ("v_stride", ctypes.c_int64 * 3),
                ("log_decay", ctypes.c_void_p), ("start", ctypes.c_void_p), ("start_stride", ctypes.c_int64 * 2),
                ("state", ctypes.c_void_p), ("scale", ctypes.c_float)]


def missing(path):
    return RuntimeError(f"{os.path.basename(path)} not built ({path}); run __graft_entry__.build() -- no CPU fallback exists")


def lib():
    """The loaded library; RuntimeError if it is not built."""
    global _lib
    if _lib is None:
        import torch  # noqa: F401  (its HIP runtime has to be the process' one: loaded first)
        if not os.path.exists(LIB_PATH):
            raise missing(LIB_PATH)
        L = ctypes.CDLL(LIB_PATH)
        P, I, Q, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
        L.urgym_ops_last_error.restype = ctypes.c_char_p
        L.urgym_ops_layer_norm.argtypes = [I, I, Q, Q, P, Q, P, P, F, P, P, P, P]
        L.urgym_ops_layer_norm_workspace.argtypes = [Q, Q]
        L.urgym_ops_layer_norm_workspace.restype = Q
        L.urgym_ops_layer_norm_backward.argtypes = [I, I, Q, Q, P, Q, P, Q, P, P, P, P, P, P, P, P]
        L.urgym_ops_decay_workspace.argtypes = [ctypes.POINTER(Seq)]
        L.urgym_ops_decay_backward_workspace.argtypes = [ctypes.POINTER(Seq), P, Q * 3]
        L.urgym_ops_decay_workspace.restype = L.urgym_ops_decay_backward_workspace.restype = Q
        L.urgym_ops_decay.argtypes = [ctypes.POINTER(Seq), P, P, P, P]
        L.urgym_ops_decay_backward.argtypes = [ctypes.POINTER(Seq), P, Q * 3, P, P, P, P, P, P, P]
        L.urgym_ops_decay_step.argtypes = [I, Q, I, I, I, P, Q, Q, P, Q, Q, P, Q, Q, P, P, Q, F, P, P, P, P]
        _lib = L
    return _lib
