"""ctypes binding of libisa_block_hip.so (declared in include/isa_block.h).

As for the FFN's library, it is the only compute path: loading fails loudly when it is missing
or was built for another ABI, and torch is imported first so that both use one HIP runtime.
"""

from __future__ import annotations

import ctypes
import threading
from pathlib import Path

import torch

from isa.kernels.transformer_ffn._hip import HipExtensionError, on_device, stream_handle  # noqa: F401

ABI_VERSION = 1
LIB_NAME = "libisa_block_hip.so"
LIB_PATH = Path(__file__).resolve().parent / LIB_NAME

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
REDUCTIONS = {"mean": 0, "sum": 1, "none": 2}
NORM_MAX_DIM = 16384
ATTENTION_MAX_DIM = 128

EXPORTS = (
    "isa_block_abi_version",
    "isa_block_last_error",
    "isa_block_norm_forward",
    "isa_block_norm_backward_workspace",
    "isa_block_norm_backward",
    "isa_block_attention_forward_workspace",
    "isa_block_attention_forward",
    "isa_block_attention_backward_workspace",
    "isa_block_attention_backward",
    "isa_block_loss_workspace",
    "isa_block_loss_forward",
    "isa_block_loss_backward",
    "isa_block_loss_with_grad",
)

_vp, _i64, _int, _f32, _size = (ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_size_t)


class Norm(ctypes.Structure):
    """isa_block_norm."""

    _fields_ = [("type", _int), ("x_type", _int), ("weight_type", _int), ("rows", _i64), ("dim", _i64),
                ("eps", _f32), ("weight", _vp), ("bias", _vp)]


class Attention(ctypes.Structure):
    """isa_block_attention."""

    _fields_ = [("type", _int), ("batch", _i64), ("queries", _i64), ("keys", _i64), ("heads", _i64),
                ("kv_heads", _i64), ("head_dim", _i64), ("window", _i64), ("sinks", _i64), ("scale", _f32),
                ("key_lengths", _vp), ("q", _vp), ("k", _vp), ("v", _vp), ("q_strides", _i64 * 3),
                ("k_strides", _i64 * 3), ("v_strides", _i64 * 3)]


class Loss(ctypes.Structure):
    """isa_block_loss."""

    _fields_ = [("type", _int), ("rows", _i64), ("vocab", _i64), ("ignore_index", _i64), ("logits", _vp),
                ("logits_stride", _i64), ("targets", _vp)]


_lock = threading.Lock()
_lib = None


def _declare(lib) -> None:
    norm, att, loss = (ctypes.POINTER(t) for t in (Norm, Attention, Loss))

    def declare(name, result, *arguments):
        f = getattr(lib, name)
        f.restype, f.argtypes = result, list(arguments)

    declare("isa_block_abi_version", _int)
    declare("isa_block_last_error", ctypes.c_char_p)
    declare("isa_block_norm_forward", _int, norm, _vp, _i64, _vp, _i64, _vp, _vp, _vp, _vp, _vp)
    declare("isa_block_norm_backward_workspace", _size, _i64, _i64)
    declare("isa_block_norm_backward", _int, norm, _vp, _vp, _vp, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _size, _vp)
    declare("isa_block_attention_forward_workspace", _size, att)
    declare("isa_block_attention_forward", _int, att, _vp, _vp, _vp, _vp, _size, _vp)
    declare("isa_block_attention_backward_workspace", _size, att)
    declare("isa_block_attention_backward", _int, att, _vp, _vp, _vp, _vp, ctypes.POINTER(_i64), _vp, _vp, _vp, _vp,
            _size, _vp)
    declare("isa_block_loss_workspace", _size, loss)
    declare("isa_block_loss_forward", _int, loss, _int, _vp, _vp, _vp, _vp, _size, _vp)
    declare("isa_block_loss_backward", _int, loss, _int, _vp, _vp, _vp, _vp, _i64, _vp)
    declare("isa_block_loss_with_grad", _int, loss, _f32, _vp, _vp, _i64, _vp, _size, _vp)


def load(path: Path | None = None):
    """Load and cache the library; raise HipExtensionError if it is absent or mismatched."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        p = Path(path) if path is not None else LIB_PATH
        if not p.exists():
            raise HipExtensionError(f"{LIB_NAME} not found at {p}; build it with `python isa-_amd/csrc/build.py` "
                                    "(or __graft_entry__.build())")
        lib = ctypes.CDLL(str(p))
        missing = [name for name in EXPORTS if not hasattr(lib, name)]
        if missing:
            raise HipExtensionError(f"{p} lacks exports {missing}")
        _declare(lib)
        version = lib.isa_block_abi_version()
        if version != ABI_VERSION:
            raise HipExtensionError(f"{p} has ABI version {version}, expected {ABI_VERSION}; rebuild it")
        _lib = lib
        return lib


def check(rc: int, what: str) -> None:
    """Raise RuntimeError carrying the library's message for a nonzero status."""
    if rc != 0:
        msg = load().isa_block_last_error()
        raise RuntimeError(f"{what} failed ({rc}): {msg.decode('utf-8', 'replace') if msg else ''}")
