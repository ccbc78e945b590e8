"""The block's C ABI loads on a host without a GPU, exports what include/isa_block.h declares and
refuses bad arguments before any HIP call (CPU only: no kernel is launched here)."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

from isa.kernels.transformer_block import _hip

HEADER = Path(__file__).resolve().parents[1] / "include" / "isa_block.h"
FAKE = ctypes.c_void_p(4096)  # never dereferenced: validation fails first


def declared_functions():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    return sorted(set(re.findall(r"\b(isa_block_\w+)\s*\(", text)))


def test_header_lists_the_python_exports():
    assert declared_functions() == sorted(_hip.EXPORTS)


def test_library_exports_every_declared_symbol():
    raw = ctypes.CDLL(str(_hip.LIB_PATH))
    for name in declared_functions():
        assert hasattr(raw, name), name
    assert raw.isa_block_abi_version() == _hip.ABI_VERSION


def test_missing_library_is_refused(tmp_path, monkeypatch):
    monkeypatch.setattr(_hip, "_lib", None)
    with pytest.raises(_hip.HipExtensionError, match="not found"):
        _hip.load(tmp_path / "absent.so")


def refused(rc, text):
    message = _hip.load().isa_block_last_error().decode()
    assert rc == -1 and text in message, (rc, message)


def norm(**over):
    n = _hip.Norm(0, 0, 0, 4, 64, 1e-5, 4096, None)
    for k, v in over.items():
        setattr(n, k, v)
    return ctypes.byref(n)


def test_norm_refusals():
    lib = _hip.load()

    def forward(x=None, h=None, y=FAKE, mean=None, rstd=None, **over):
        return lib.isa_block_norm_forward(norm(**over), x, 64, FAKE, 64, y, h, mean, rstd, None)

    refused(lib.isa_block_norm_forward(None, None, 0, FAKE, 64, FAKE, None, None, None, None), "null")
    refused(forward(type=7), "type")
    refused(forward(type=1, x_type=0, weight_type=1), "x has")
    refused(forward(weight_type=1), "weight has")
    refused(forward(rows=-1), "negative rows")
    refused(forward(dim=0), "dim")
    refused(forward(dim=16385), "16384")
    refused(forward(eps=-1.0), "eps")
    refused(forward(weight=None), "weight")
    refused(forward(y=None), "must be set")
    refused(forward(x=FAKE), "go together")
    refused(forward(mean=FAKE), "go together")
    refused(forward(x_type=1), "without x")
    assert forward(rows=0) == 0

    def backward(dy=FAKE, dx=None, dw=FAKE, db=FAKE, ws=FAKE, size=1 << 30, **over):
        return lib.isa_block_norm_backward(norm(**over), dy, None, FAKE, 64, FAKE, FAKE, dx, FAKE, dw, db, ws, size, None)

    refused(backward(dy=None), "must be set")
    refused(backward(dx=FAKE), "grad_x")
    refused(backward(x_type=1), "grad_x")
    refused(backward(dw=None), "grad_weight")
    refused(backward(size=16), "workspace too small")
    refused(backward(ws=ctypes.c_void_p(4100)), "aligned")
    assert backward(rows=0, dw=None, db=None) == 0
    assert lib.isa_block_norm_backward_workspace(-1, 64) == 0
    assert lib.isa_block_norm_backward_workspace(8192, 768) >= 2 * 768 * 4


def attention(**over):
    a = _hip.Attention()
    a.type, a.batch, a.queries, a.keys, a.heads, a.kv_heads, a.head_dim = 1, 2, 8, 8, 4, 2, 64
    a.scale = 0.125
    a.q = a.k = a.v = 4096
    for name, heads in (("q_strides", 4), ("k_strides", 2), ("v_strides", 2)):
        getattr(a, name)[:] = (8 * heads * 64, heads * 64, 64)
    for k, v in over.items():
        if k.endswith("strides"):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return ctypes.byref(a)


def test_attention_refusals():
    lib = _hip.load()

    def forward(out=FAKE, ws=FAKE, size=1 << 40, **over):
        return lib.isa_block_attention_forward(attention(**over), out, None, None, ws, size, None)

    refused(lib.isa_block_attention_forward(None, FAKE, None, None, None, 0, None), "null")
    refused(forward(type=3), "type")
    refused(forward(queries=-1), "sizes")
    refused(forward(keys=1 << 31), "sizes")
    refused(forward(window=-1), "sizes")
    refused(forward(heads=3), "multiple of kv_heads")
    refused(forward(kv_heads=0), "kv_heads")
    refused(forward(head_dim=12), "head_dim")
    refused(forward(head_dim=136), "head_dim")
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        refused(forward(scale=scale), "scale")
    refused(forward(q=None), "q is null")
    refused(forward(k=None), "k and v")
    refused(forward(v=4100), "aligned")
    refused(forward(k_strides=(1024, 129, 64)), "strides")
    refused(forward(out=None), "out must be set")
    refused(forward(out=ctypes.c_void_p(4104)), "aligned")
    refused(forward(batch=1 << 20, queries=1 << 20, keys=1), "too many rows")
    assert forward(batch=0) == 0 and forward(queries=0) == 0

    strides = (ctypes.c_int64 * 3)(8 * 4 * 64, 4 * 64, 64)

    def backward(out=FAKE, lse=FAKE, dout=FAKE, dq=FAKE, dk=FAKE, dv=FAKE, ws=FAKE, size=1 << 40, by=strides, **over):
        return lib.isa_block_attention_backward(attention(**over), out, None, lse, dout, by, dq, dk, dv, ws, size, None)

    refused(backward(lse=None), "must be set")
    refused(backward(by=None), "must be set")
    refused(backward(dk=None), "go together")
    refused(backward(dout=ctypes.c_void_p(4100)), "aligned")
    refused(backward(by=(ctypes.c_int64 * 3)(8 * 4 * 64, 4, 64)), "strides")
    refused(backward(size=16), "workspace too small")
    refused(backward(ws=ctypes.c_void_p(4100)), "aligned")
    refused(backward(dq=ctypes.c_void_p(4100)), "aligned")
    assert backward(batch=0) == 0
    assert lib.isa_block_attention_backward_workspace(attention(head_dim=7)) == 0
    assert lib.isa_block_attention_backward_workspace(attention()) >= 2 * 4 * 8 * 4


def loss(**over):
    n = _hip.Loss(0, 4, 100, -100, 4096, 100, 4096)
    for k, v in over.items():
        setattr(n, k, v)
    return ctypes.byref(n)


def test_loss_refusals():
    lib = _hip.load()

    def with_grad(out=FAKE, grad=FAKE, ws=FAKE, size=1 << 30, **over):
        return lib.isa_block_loss_with_grad(loss(**over), 1.0, out, grad, 100, ws, size, None)

    refused(lib.isa_block_loss_with_grad(None, 1.0, FAKE, FAKE, 1, FAKE, 0, None), "null")
    refused(with_grad(type=-1), "type")
    refused(with_grad(rows=-1), "rows")
    refused(with_grad(rows=(1 << 24) + 1), "rows")
    refused(with_grad(vocab=0), "vocab")
    refused(with_grad(logits=None), "must be set")
    refused(with_grad(targets=None), "must be set")
    refused(with_grad(logits=4098), "aligned")
    refused(with_grad(out=None), "must be set")
    refused(with_grad(grad=None), "must be set")
    refused(with_grad(grad=ctypes.c_void_p(4098)), "aligned")
    refused(with_grad(size=0), "workspace too small")
    refused(with_grad(ws=ctypes.c_void_p(4100)), "aligned")

    def forward(reduction=0, out=FAKE, size=1 << 30, **over):
        return lib.isa_block_loss_forward(loss(**over), reduction, out, None, None, FAKE, size, None)

    refused(forward(reduction=3), "reduction")
    refused(forward(out=None), "out is null")
    refused(forward(size=0), "workspace too small")
    assert forward(reduction=2, rows=0) == 0

    def backward(reduction=0, stats=FAKE, count=FAKE, up=FAKE, grad=FAKE, **over):
        return lib.isa_block_loss_backward(loss(**over), reduction, stats, count, up, grad, 100, None)

    refused(backward(reduction=-1), "reduction")
    refused(backward(stats=None), "must be set")
    refused(backward(count=None), "must be set")
    refused(backward(up=None), "must be set")
    refused(backward(grad=ctypes.c_void_p(4097)), "aligned")
    assert backward(rows=0) == 0


def test_cpu_tensors_are_refused():
    from isa.kernels.transformer_block import (add_layer_norm, cross_entropy, cross_entropy_with_grad, layer_norm,
                                               window_attention)

    x, w = torch.zeros(2, 8), torch.ones(8)
    q = torch.zeros(1, 2, 1, 8)
    for call in (lambda: layer_norm(x, w), lambda: add_layer_norm(x, x, w), lambda: window_attention(q, q, q),
                 lambda: cross_entropy(x, torch.zeros(2, dtype=torch.int64)),
                 lambda: cross_entropy_with_grad(x, torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
