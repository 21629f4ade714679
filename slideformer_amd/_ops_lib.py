"""ctypes binding of ``libslideformer_amd_ops.so`` (C-ABI declared in ``include/model_ops.h``).

Loaded after ``import torch``, like the optimizer's library, and with no fallback:
if it is missing, ``load()`` raises.
"""
from __future__ import annotations

import ctypes
import importlib.util
import os
import threading

import torch  # noqa: F401  (binds the HIP runtime before the library is loaded)

from . import _lib

# where slideformer_amd/build.py writes the library
LIB_PATH = os.path.join(os.path.dirname(_lib.LIB_PATH), "libslideformer_amd_ops.so")

# where it writes the native host module
CALLS_PATH = os.path.join(os.path.dirname(LIB_PATH), "_ops_calls.so")

# LA_OPS_ABI_VERSION of include/model_ops.h that these bindings declare
ABI_VERSION = 1

LA_I32, LA_I64, LA_I8, LA_F8E4M3 = 16, 17, 18, 19

# every exported symbol of include/model_ops.h
EXPORTED = (
    "la_ops_abi_version",
    "la_embedding",
    "la_embedding_grad_workspace",
    "la_embedding_grad",
    "la_rms_norm",
    "la_rms_norm_grad_workspace",
    "la_rms_norm_grad",
    "la_linear_loss_workspace",
    "la_linear_loss",
)


class LaLinearLoss(ctypes.Structure):
    """Mirror of ``la_linear_loss_t``."""

    _fields_ = [
        ("dtype", ctypes.c_int),
        ("x", ctypes.c_void_p),
        ("n", ctypes.c_uint64),
        ("hidden", ctypes.c_uint64),
        ("x_stride", ctypes.c_uint64),
        ("weight", ctypes.c_void_p),
        ("vocab", ctypes.c_uint64),
        ("weight_stride", ctypes.c_uint64),
        ("targets", ctypes.c_void_p),
        ("ignore_index", ctypes.c_int64),
        ("mean", ctypes.c_int),
        ("loss", ctypes.c_void_p),
        ("row_loss", ctypes.c_void_p),
        ("grads", ctypes.c_int),
        ("grad_scale", ctypes.c_void_p),
        ("grad_x", ctypes.c_void_p),
        ("grad_x_stride", ctypes.c_uint64),
        ("grad_weight_dtype", ctypes.c_int),
        ("grad_weight", ctypes.c_void_p),
        ("grad_weight_stride", ctypes.c_uint64),
        ("accumulate", ctypes.c_int),
        ("piece_rows", ctypes.c_uint64),
    ]


_lock = threading.Lock()
_loaded = None


def _declare(L):
    P = ctypes.c_void_p
    f, i, u64, i64 = ctypes.c_float, ctypes.c_int, ctypes.c_uint64, ctypes.c_int64
    call = ctypes.POINTER(LaLinearLoss)
    L.la_ops_abi_version.argtypes = []
    L.la_ops_abi_version.restype = i
    L.la_embedding.argtypes = [i, P, u64, i, P, u64, u64, u64, f, P, u64, P]
    L.la_embedding.restype = i
    L.la_embedding_grad_workspace.argtypes = [u64, u64, u64]
    L.la_embedding_grad_workspace.restype = u64
    L.la_embedding_grad.argtypes = [i, P, u64, i, P, u64, i, P, u64, u64, u64, f, i64, i, P, u64, P]
    L.la_embedding_grad.restype = i
    L.la_rms_norm.argtypes = [i, P, u64, P, u64, P, u64, u64, f, P, u64, i, P, u64, P, P, P]
    L.la_rms_norm.restype = i
    L.la_rms_norm_grad_workspace.argtypes = [u64, u64]
    L.la_rms_norm_grad_workspace.restype = u64
    L.la_rms_norm_grad.argtypes = [i, P, u64, P, u64, P, P, P, u64, u64, u64, P, u64, i, P, i, P, u64, P]
    L.la_rms_norm_grad.restype = i
    L.la_linear_loss_workspace.argtypes = [call]
    L.la_linear_loss_workspace.restype = u64
    L.la_linear_loss.argtypes = [call, P, u64, P]
    L.la_linear_loss.restype = i
    return L


def load():
    """Load the HIP library (once).  Raises ImportError if it has not been built."""
    global _loaded
    if _loaded is not None:
        return _loaded
    with _lock:
        if _loaded is None:
            if not os.path.exists(LIB_PATH):
                raise ImportError(f"slideformer_amd HIP library not found at {LIB_PATH}; build it with "
                                  "`python -m slideformer_amd.build` (there is no CPU fallback)")
            raw = ctypes.CDLL(LIB_PATH)
            raw.la_ops_abi_version.restype = ctypes.c_int
            found = raw.la_ops_abi_version()
            if found != ABI_VERSION:
                raise ImportError(f"{LIB_PATH} implements the C-ABI version {found}, this package needs "
                                  f"{ABI_VERSION}; rebuild it with `python -m slideformer_amd.build`")
            _loaded = _declare(raw)
        return _loaded


_calls = None


def calls():
    """The native host module (csrc/ops_calls.cpp), bound once to the loaded
    library.  Raises ImportError if it has not been built."""
    global _calls
    if _calls is None:
        L = load()
        with _lock:
            if _calls is None:
                if not os.path.exists(CALLS_PATH):
                    raise ImportError(f"{CALLS_PATH} not found; build it with `python -m slideformer_amd.build`")
                spec = importlib.util.spec_from_file_location("_ops_calls", CALLS_PATH)
                module = importlib.util.module_from_spec(spec)
                spec.loader.exec_module(module)
                module.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
                    L.la_embedding, L.la_embedding_grad_workspace, L.la_embedding_grad, L.la_rms_norm,
                    L.la_rms_norm_grad_workspace, L.la_rms_norm_grad)))
                _calls = module
    return _calls
