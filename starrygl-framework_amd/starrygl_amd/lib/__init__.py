"""Loader of libsgl_hot.so, the HIP implementation of include/sgl_hot.h.

There is no CPU fallback: if the shared library is missing, `load()` raises.
PyTorch is imported first so that the library binds to the HIP runtime that
PyTorch already mapped (one runtime per process, shared streams and pointers).
"""
import ctypes as C
import os

from . import _abi

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libsgl_hot.so")

_lib = None


def load():
    """-> bound entry points of libsgl_hot.so (loaded once per process)."""
    global _lib
    if _lib is None:
        import torch  # noqa: F401  (maps libamdhip64 before our library needs it)
        if not os.path.exists(LIB_PATH):
            raise ImportError(
                f"{LIB_PATH} is missing: build it with `make -C starrygl-framework_amd/csrc` "
                "(or __graft_entry__.build()); this package has no CPU fallback")
        _lib = _abi.bind(C.CDLL(LIB_PATH), "sgl_")
    return _lib


_torch_ops = None


def torch_ops():
    """-> the compiled autograd side of the attention-layer operators (csrc/torch_ops.cpp), driving `load()`'s library."""
    global _torch_ops
    if _torch_ops is None:
        lib = load()
        try:
            from . import sgl_torch
        except ImportError as e:
            raise ImportError(f"sgl_torch.so is missing or does not load ({e}): build it with `make -C starrygl-framework_amd/csrc` "
                              "(or __graft_entry__.build())") from e
        names = ("last_error_string", "rotary", "qk_norm_rotary", "qk_norm_rotary_backward_workspace_bytes",
                 "qk_norm_rotary_backward", "diff_attn_workspace_bytes", "diff_attn", "diff_attn_backward_workspace_bytes",
                 "diff_attn_backward")
        sgl_torch.init([C.cast(getattr(lib, n), C.c_void_p).value for n in names])
        _torch_ops = sgl_torch
    return _torch_ops


_hot = {}


def hot_path(device="cuda:0"):
    """-> HotPath driving libsgl_hot.so on `device` (cached per device)."""
    import torch
    from .driver import HotPath, TorchBackend
    dev = torch.device(device)
    if dev.type != "cuda":
        raise RuntimeError("the sgl hot path runs on a HIP device only (got %s)" % dev)
    if dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    key = str(dev)
    if key not in _hot:
        _hot[key] = HotPath(load(), TorchBackend(dev))
    return _hot[key]
