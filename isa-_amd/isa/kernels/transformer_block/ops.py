"""Tensor-level calls into libisa_block_hip.so.

Every function checks on the host what the kernels assume (device, types, shapes, strides,
alignment), allocates outputs and workspace with the caching allocator and enqueues on the
current stream of the tensors' device. Nothing here is tracked by autograd.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from isa.kernels.transformer_block import _hip


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _require(t: torch.Tensor, name: str, device: Optional[torch.device] = None) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if t.dtype not in _hip.TYPES:
        raise RuntimeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if device is not None and t.device != device:
        raise RuntimeError(f"{name} must be on {device}, got {t.device}")


def _workspace(nbytes: int, device: torch.device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


# ---- layer norm ---------------------------------------------------------------------------


def rows_of(t: torch.Tensor) -> torch.Tensor:
    """t as [rows, dim] with adjacent elements in a row: a copy only where no view does it."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _norm(residual: torch.Tensor, x_dtype: torch.dtype, weight: torch.Tensor, bias: Optional[torch.Tensor],
          eps: float) -> "_hip.Norm":
    n = _hip.Norm()
    n.type, n.x_type, n.weight_type = _hip.TYPES[residual.dtype], _hip.TYPES[x_dtype], _hip.TYPES[weight.dtype]
    n.rows, n.dim = residual.shape
    n.eps = eps
    n.weight, n.bias = weight.data_ptr(), _ptr(bias)
    return n


def check_norm(x: Optional[torch.Tensor], residual: torch.Tensor, weight: torch.Tensor,
               bias: Optional[torch.Tensor]) -> None:
    name = "x" if x is None else "residual"
    _require(residual, name)
    dev, dtype = residual.device, residual.dtype
    if residual.dim() < 1 or not 1 <= residual.shape[-1] <= _hip.NORM_MAX_DIM:
        raise RuntimeError(f"{name}'s last dimension must be 1 to {_hip.NORM_MAX_DIM}, got shape {tuple(residual.shape)}")
    if x is not None:
        _require(x, "x", dev)
        if x.shape != residual.shape:
            raise RuntimeError(f"x and residual must have one shape, got {tuple(x.shape)} and {tuple(residual.shape)}")
        if x.dtype != dtype and dtype != torch.float32:
            raise RuntimeError(f"x must be {dtype} as residual is (or residual float32), got {x.dtype}")
    _require(weight, "weight", dev)
    if weight.dtype not in (dtype, torch.float32):
        raise RuntimeError(f"weight must be {dtype} or float32, got {weight.dtype}")
    if tuple(weight.shape) != (residual.shape[-1],):
        raise RuntimeError(f"weight must be [{residual.shape[-1]}], got {tuple(weight.shape)}")
    if bias is not None:
        _require(bias, "bias", dev)
        if bias.dtype != weight.dtype or bias.shape != weight.shape:
            raise RuntimeError("bias must have weight's type and shape")


def norm_forward(x: Optional[torch.Tensor], residual: torch.Tensor, weight: torch.Tensor,
                 bias: Optional[torch.Tensor], eps: float, with_stats: bool
                 ) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(y, h, stats) of rows [rows, dim]: h None without x, stats ([2, rows] fp32: mean, rstd) None
    unless asked for."""
    lib, dev = _hip.load(), residual.device
    n = _norm(residual, residual.dtype if x is None else x.dtype, weight, bias, eps)
    y = torch.empty(residual.shape, dtype=residual.dtype, device=dev)
    h = None if x is None else torch.empty(residual.shape, dtype=residual.dtype, device=dev)
    rows = residual.shape[0]
    stats = torch.empty((2, rows), dtype=torch.float32, device=dev) if with_stats else None
    mean = None if stats is None else stats.data_ptr()
    with _hip.on_device(dev):
        rc = lib.isa_block_norm_forward(ctypes.byref(n), _ptr(x), 0 if x is None else x.stride(0),
                                        residual.data_ptr(), residual.stride(0), y.data_ptr(), _ptr(h), mean,
                                        None if mean is None else mean + 4 * rows, _hip.stream_handle(dev))
    _hip.check(rc, "isa_block_norm_forward")
    return y, h, stats


def norm_backward(dy: torch.Tensor, dh: Optional[torch.Tensor], h: torch.Tensor, stats: torch.Tensor,
                  weight: torch.Tensor, x_dtype: torch.dtype, with_weight: bool, with_bias: bool):
    """(grad of x or None where it is the residual's, grad of residual, of weight or None, of bias or
    None) of rows [rows, dim]."""
    lib, dev = _hip.load(), h.device
    rows, dim = h.shape
    n = _norm(h, x_dtype, weight, None, 0.0)
    dy = dy.contiguous()
    dh = None if dh is None else dh.contiguous()
    dr = torch.empty((rows, dim), dtype=h.dtype, device=dev)
    dx = torch.empty((rows, dim), dtype=x_dtype, device=dev) if x_dtype != h.dtype else None
    dw = db = ws = None
    if with_weight or with_bias:
        dw = torch.empty(dim, dtype=weight.dtype, device=dev)
        db = torch.empty(dim, dtype=weight.dtype, device=dev) if with_bias else None
        ws = _workspace(lib.isa_block_norm_backward_workspace(rows, dim), dev)
    mean = stats.data_ptr()
    with _hip.on_device(dev):
        rc = lib.isa_block_norm_backward(ctypes.byref(n), dy.data_ptr(), _ptr(dh), h.data_ptr(), h.stride(0), mean,
                                         mean + 4 * rows, _ptr(dx), dr.data_ptr(), _ptr(dw), _ptr(db), _ptr(ws),
                                         0 if ws is None else ws.numel(), _hip.stream_handle(dev))
    _hip.check(rc, "isa_block_norm_backward")
    return dx, dr, dw, db


# ---- attention ------------------------------------------------------------------------------


def _strides(t: torch.Tensor):
    """Strides of batch, token and head; a dimension of one element has none that matters."""
    n, s = t.shape, t.stride()
    return tuple(s[i] if n[i] > 1 else 0 for i in range(3))


def attention_operand(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy where its heads' elements are apart, 16-byte loads would not be aligned or tokens
    overlap (as broadcast ones do) or lie too far apart."""
    if t.numel() == 0:
        return t
    s = _strides(t)
    if t.stride(3) == 1 and not t.data_ptr() & 15 and not any(x & 7 for x in s) and (
            t.shape[1] < 2 or t.shape[3] <= s[1] < _FAR // t.element_size()):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def check_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: Optional[int], sinks: int,
                    scale: Optional[float], key_lengths: Optional[torch.Tensor]) -> None:
    _require(q, "q")
    for t, name in ((k, "k"), (v, "v")):
        _require(t, name, q.device)
        if t.dtype != q.dtype:
            raise RuntimeError(f"{name} must be {q.dtype} as q is, got {t.dtype}")
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise RuntimeError("q must be [batch, queries, heads, head_dim], k and v [batch, keys, kv_heads, head_dim]; "
                           f"got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    if q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise RuntimeError(f"batch and head_dim of q {tuple(q.shape)} and k {tuple(k.shape)} differ")
    if k.shape[2] < 1 or q.shape[2] < 1 or q.shape[2] % k.shape[2]:
        raise RuntimeError(f"heads ({q.shape[2]}) must be a multiple of kv_heads ({k.shape[2]})")
    if q.shape[3] % 8 or not 8 <= q.shape[3] <= _hip.ATTENTION_MAX_DIM:
        raise RuntimeError(f"head_dim must be a multiple of 8 up to {_hip.ATTENTION_MAX_DIM}, got {q.shape[3]}")
    if window is not None and window < 1:
        raise RuntimeError(f"window must be None or at least 1, got {window}")
    if sinks < 0:
        raise RuntimeError(f"sinks must not be negative, got {sinks}")
    if scale is not None and not 0.0 < scale < math.inf:
        raise RuntimeError(f"scale must be positive and finite, got {scale}")
    if key_lengths is not None:
        if key_lengths.dtype not in (torch.int32, torch.int64) or tuple(key_lengths.shape) != (q.shape[0],):
            raise RuntimeError(f"key_lengths must be int32 or int64 [{q.shape[0]}], got {key_lengths.dtype} "
                               f"{tuple(key_lengths.shape)}")
        if key_lengths.device != q.device:
            raise RuntimeError(f"key_lengths must be on {q.device}, got {key_lengths.device}")


def _attention(q, k, v, window, sinks, scale, key_lengths) -> "_hip.Attention":
    a = _hip.Attention()
    a.type = _hip.TYPES[q.dtype]
    a.batch, a.queries, a.heads, a.head_dim = q.shape
    a.keys, a.kv_heads = k.shape[1], k.shape[2]
    a.window = min(window or 0, _LONGEST)  # past the longest sequence: no window
    a.sinks = min(sinks, _LONGEST)
    a.scale = scale
    a.key_lengths = _ptr(key_lengths)
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.q_strides[:], a.k_strides[:], a.v_strides[:] = _strides(q), _strides(k), _strides(v)
    return a


_LONGEST = 1 << 30
_FAR = 1 << 24  # bytes between tokens


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: Optional[int], sinks: int,
                      scale: float, key_lengths: Optional[torch.Tensor], for_backward: bool):
    """(out, rest, lse): the latter two for a backward call, else None; rest (what out's rounding left)
    in 16-bit types only. Operands from attention_operand(), key_lengths int32."""
    lib, dev = _hip.load(), q.device
    a = _attention(q, k, v, window, sinks, scale, key_lengths)
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    lse = torch.empty((q.shape[0], q.shape[2], q.shape[1], 2), dtype=torch.float32, device=dev) if for_backward else None
    rest = torch.empty_like(out) if for_backward and q.dtype != torch.float32 else None
    ws = _workspace(lib.isa_block_attention_forward_workspace(ctypes.byref(a)), dev)
    with _hip.on_device(dev):
        rc = lib.isa_block_attention_forward(ctypes.byref(a), out.data_ptr(), _ptr(rest), _ptr(lse),
                                             _ptr(ws), 0 if ws is None else ws.numel(), _hip.stream_handle(dev))
    _hip.check(rc, "isa_block_attention_forward")
    return out, rest, lse


def attention_backward(q, k, v, out, rest, lse, dout, window, sinks, scale, key_lengths, with_q: bool = True,
                       with_kv: bool = True):
    """(grad of q or None, grads of k and v or None)."""
    lib, dev = _hip.load(), q.device
    a = _attention(q, k, v, window, sinks, scale, key_lengths)
    dout = attention_operand(dout)
    dq = torch.empty(q.shape, dtype=q.dtype, device=dev) if with_q else None
    dk = torch.empty(k.shape, dtype=k.dtype, device=dev) if with_kv else None
    dv = torch.empty(v.shape, dtype=v.dtype, device=dev) if with_kv else None
    ws = _workspace(lib.isa_block_attention_backward_workspace(ctypes.byref(a)), dev)
    with _hip.on_device(dev):
        rc = lib.isa_block_attention_backward(ctypes.byref(a), out.data_ptr(), _ptr(rest), lse.data_ptr(),
                                              dout.data_ptr(), (ctypes.c_int64 * 3)(*_strides(dout)), _ptr(dq), _ptr(dk), _ptr(dv),
                                              _ptr(ws), 0 if ws is None else ws.numel(), _hip.stream_handle(dev))
    _hip.check(rc, "isa_block_attention_backward")
    return dq, dk, dv


# ---- cross-entropy ------------------------------------------------------------------------


def check_loss(logits: torch.Tensor, targets: torch.Tensor) -> None:
    _require(logits, "logits")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise RuntimeError(f"logits must be [..., vocab], got {tuple(logits.shape)}")
    if targets.dtype != torch.int64 or targets.shape != logits.shape[:-1]:
        raise RuntimeError(f"targets must be int64 {tuple(logits.shape[:-1])}, got {targets.dtype} "
                           f"{tuple(targets.shape)}")
    if targets.device != logits.device:
        raise RuntimeError(f"targets must be on {logits.device}, got {targets.device}")


def _loss(logits: torch.Tensor, targets: torch.Tensor, ignore_index: int) -> "_hip.Loss":
    n = _hip.Loss()
    n.type = _hip.TYPES[logits.dtype]
    n.rows, n.vocab = logits.shape
    n.ignore_index = ignore_index
    n.logits, n.logits_stride, n.targets = logits.data_ptr(), logits.stride(0), targets.data_ptr()
    return n


def like_rows(t: torch.Tensor) -> torch.Tensor:
    """A new tensor as t [rows, vocab], its rows as far apart (so both are aligned alike)."""
    rows, dim = t.shape
    stride = t.stride(0)
    if rows < 2 or stride <= dim:
        return torch.empty((rows, dim), dtype=t.dtype, device=t.device)
    return torch.empty_strided((rows, dim), (stride, 1), dtype=t.dtype, device=t.device)


def loss_forward(logits: torch.Tensor, targets: torch.Tensor, ignore_index: int, reduction: str, with_stats: bool):
    """(loss, stats [rows, 2] or None, count [1] or None) of logits [rows, vocab]."""
    lib, dev = _hip.load(), logits.device
    n = _loss(logits, targets, ignore_index)
    rows = logits.shape[0]
    out = torch.empty((rows,) if reduction == "none" else (), dtype=torch.float32, device=dev)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=dev) if with_stats else None
    count = torch.empty(1, dtype=torch.float32, device=dev) if with_stats else None
    ws = _workspace(lib.isa_block_loss_workspace(ctypes.byref(n)), dev)
    with _hip.on_device(dev):
        rc = lib.isa_block_loss_forward(ctypes.byref(n), _hip.REDUCTIONS[reduction], out.data_ptr(), _ptr(stats),
                                        _ptr(count), ws.data_ptr(), ws.numel(), _hip.stream_handle(dev))
    _hip.check(rc, "isa_block_loss_forward")
    return out, stats, count


def loss_backward(logits, targets, ignore_index: int, reduction: str, stats, count, grad_out) -> torch.Tensor:
    lib, dev = _hip.load(), logits.device
    n = _loss(logits, targets, ignore_index)
    grad = like_rows(logits)
    grad_out = grad_out.to(torch.float32).contiguous()
    with _hip.on_device(dev):
        rc = lib.isa_block_loss_backward(ctypes.byref(n), _hip.REDUCTIONS[reduction], stats.data_ptr(),
                                         count.data_ptr(), grad_out.data_ptr(), grad.data_ptr(), grad.stride(0),
                                         _hip.stream_handle(dev))
    _hip.check(rc, "isa_block_loss_backward")
    return grad


def loss_with_grad(logits: torch.Tensor, targets: torch.Tensor, ignore_index: int, grad_scale: float):
    """(mean loss, grad_scale times its gradient) of logits [rows, vocab]."""
    lib, dev = _hip.load(), logits.device
    n = _loss(logits, targets, ignore_index)
    out = torch.empty((), dtype=torch.float32, device=dev)
    grad = like_rows(logits)
    ws = _workspace(lib.isa_block_loss_workspace(ctypes.byref(n)), dev)
    with _hip.on_device(dev):
        rc = lib.isa_block_loss_with_grad(ctypes.byref(n), grad_scale, out.data_ptr(), grad.data_ptr(),
                                          grad.stride(0), ws.data_ptr(), ws.numel(), _hip.stream_handle(dev))
    _hip.check(rc, "isa_block_loss_with_grad")
    return out, grad
