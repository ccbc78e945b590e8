"""The block's C ABI loads on a host without a GPU, exports what include/isa_block.h declares and
refuses bad arguments before any HIP call (CPU only: no kernel is launched here)."""

from __future__ import annotations

import ctypes
import re
import sys
from pathlib import Path

import pytest
import torch

from isa.kernels.transformer_block import _hip

HEADER = Path(__file__).resolve().parents[1] / "include" / "isa_block.h"
FAKE = ctypes.c_void_p(4096)  # never dereferenced: validation fails first
VP, I64, INT, F32, SIZE = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_size_t


class Norm(ctypes.Structure):
    _fields_ = [("type", INT), ("x_type", INT), ("weight_type", INT), ("rows", I64), ("dim", I64), ("eps", F32),
                ("weight", VP), ("bias", VP)]


class Attention(ctypes.Structure):
    _fields_ = [("type", INT), ("batch", I64), ("queries", I64), ("keys", I64), ("heads", I64), ("kv_heads", I64),
                ("head_dim", I64), ("window", I64), ("sinks", I64), ("scale", F32), ("key_lengths", VP), ("q", VP),
                ("k", VP), ("v", VP), ("q_strides", I64 * 3), ("k_strides", I64 * 3), ("v_strides", I64 * 3)]


class Loss(ctypes.Structure):
    _fields_ = [("type", INT), ("rows", I64), ("vocab", I64), ("ignore_index", I64), ("logits", VP),
                ("logits_stride", I64), ("targets", VP)]


NORM, ATT, LOSS = (ctypes.POINTER(t) for t in (Norm, Attention, Loss))
SIGNATURES = {
    "isa_block_abi_version": (INT,),
    "isa_block_last_error": (ctypes.c_char_p,),
    "isa_block_norm_forward": (INT, NORM, VP, I64, VP, I64, VP, VP, VP, VP, VP),
    "isa_block_norm_backward_workspace": (SIZE, I64, I64),
    "isa_block_norm_backward": (INT, NORM, VP, VP, VP, I64, VP, VP, VP, VP, VP, VP, VP, SIZE, VP),
    "isa_block_attention_forward_workspace": (SIZE, ATT),
    "isa_block_attention_forward": (INT, ATT, VP, VP, VP, VP, SIZE, VP),
    "isa_block_attention_backward_workspace": (SIZE, ATT),
    "isa_block_attention_backward": (INT, ATT, VP, VP, VP, VP, ctypes.POINTER(I64), VP, VP, VP, VP, SIZE, VP),
    "isa_block_loss_workspace": (SIZE, LOSS),
    "isa_block_loss_forward": (INT, LOSS, INT, VP, VP, VP, VP, SIZE, VP),
    "isa_block_loss_backward": (INT, LOSS, INT, VP, VP, VP, VP, I64, VP),
    "isa_block_loss_with_grad": (INT, LOSS, F32, VP, VP, I64, VP, SIZE, VP),
}


@pytest.fixture(scope="module", name="lib")
def _lib():
    lib = ctypes.CDLL(str(_hip.LIB_PATH))
    for name, (result, *arguments) in SIGNATURES.items():
        f = getattr(lib, name)
        f.restype, f.argtypes = result, arguments
    return lib


def test_header_declares_what_the_library_exports(lib):
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    assert sorted(set(re.findall(r"\b(isa_block_\w+)\s*\(", text))) == sorted(SIGNATURES)
    version = int(re.search(r"#define ISA_BLOCK_ABI_VERSION (\d+)", text).group(1))
    assert lib.isa_block_abi_version() == version == _hip.load().ABI_VERSION


def test_missing_binding_is_refused(monkeypatch):
    import isa.kernels.transformer_block as package

    monkeypatch.delattr(package, "_binding", raising=False)
    monkeypatch.setitem(sys.modules, "isa.kernels.transformer_block._binding", None)
    with pytest.raises(_hip.HipExtensionError, match="cannot be loaded"):
        _hip.load()


def refused(lib, rc, text):
    message = lib.isa_block_last_error().decode()
    assert rc == -1 and text in message, (rc, message)


def norm(**over):
    n = Norm(0, 0, 0, 4, 64, 1e-5, 4096, None)
    for k, v in over.items():
        setattr(n, k, v)
    return ctypes.byref(n)


def test_norm_refusals(lib):
    def forward(x=None, h=None, y=FAKE, mean=None, rstd=None, **over):
        return lib.isa_block_norm_forward(norm(**over), x, 64, FAKE, 64, y, h, mean, rstd, None)

    refused(lib, lib.isa_block_norm_forward(None, None, 0, FAKE, 64, FAKE, None, None, None, None), "null")
    refused(lib, forward(type=7), "type")
    refused(lib, forward(type=1, x_type=0, weight_type=1), "x has")
    refused(lib, forward(weight_type=1), "weight has")
    refused(lib, forward(rows=-1), "negative rows")
    refused(lib, forward(dim=0), "dim")
    refused(lib, forward(dim=16385), "16384")
    refused(lib, forward(eps=-1.0), "eps")
    refused(lib, forward(weight=None), "weight")
    refused(lib, forward(y=None), "must be set")
    refused(lib, forward(x=FAKE), "go together")
    refused(lib, forward(mean=FAKE), "go together")
    refused(lib, forward(x_type=1), "without x")
    assert forward(rows=0) == 0

    def backward(dy=FAKE, dx=None, dw=FAKE, db=FAKE, ws=FAKE, size=1 << 30, **over):
        return lib.isa_block_norm_backward(norm(**over), dy, None, FAKE, 64, FAKE, FAKE, dx, FAKE, dw, db, ws, size, None)

    refused(lib, backward(dy=None), "must be set")
    refused(lib, backward(dx=FAKE), "grad_x")
    refused(lib, backward(x_type=1), "grad_x")
    refused(lib, backward(dw=None), "grad_weight")
    refused(lib, backward(size=16), "workspace too small")
    refused(lib, backward(ws=ctypes.c_void_p(4100)), "aligned")
    assert backward(rows=0, dw=None, db=None) == 0
    assert lib.isa_block_norm_backward_workspace(-1, 64) == 0
    assert lib.isa_block_norm_backward_workspace(8192, 768) >= 2 * 768 * 4


def attention(**over):
    a = Attention()
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


def test_attention_refusals(lib):
    def forward(out=FAKE, ws=FAKE, size=1 << 40, **over):
        return lib.isa_block_attention_forward(attention(**over), out, None, None, ws, size, None)

    refused(lib, lib.isa_block_attention_forward(None, FAKE, None, None, None, 0, None), "null")
    refused(lib, forward(type=3), "type")
    refused(lib, forward(queries=-1), "sizes")
    refused(lib, forward(keys=1 << 31), "sizes")
    refused(lib, forward(window=-1), "sizes")
    refused(lib, forward(heads=3), "multiple of kv_heads")
    refused(lib, forward(kv_heads=0), "kv_heads")
    refused(lib, forward(head_dim=12), "head_dim")
    refused(lib, forward(head_dim=136), "head_dim")
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        refused(lib, forward(scale=scale), "scale")
    refused(lib, forward(q=None), "q is null")
    refused(lib, forward(k=None), "k and v")
    refused(lib, forward(v=4100), "aligned")
    refused(lib, forward(k_strides=(1024, 129, 64)), "strides")
    refused(lib, forward(out=None), "out must be set")
    refused(lib, forward(out=ctypes.c_void_p(4104)), "aligned")
    refused(lib, forward(batch=1 << 20, queries=1 << 20, keys=1), "too many rows")
    assert forward(batch=0) == 0 and forward(queries=0) == 0

    strides = (ctypes.c_int64 * 3)(8 * 4 * 64, 4 * 64, 64)

    def backward(out=FAKE, lse=FAKE, dout=FAKE, dq=FAKE, dk=FAKE, dv=FAKE, ws=FAKE, size=1 << 40, by=strides, **over):
        return lib.isa_block_attention_backward(attention(**over), out, None, lse, dout, by, dq, dk, dv, ws, size, None)

    refused(lib, backward(lse=None), "must be set")
    refused(lib, backward(by=None), "must be set")
    refused(lib, backward(dk=None), "go together")
    refused(lib, backward(dout=ctypes.c_void_p(4100)), "aligned")
    refused(lib, backward(by=(ctypes.c_int64 * 3)(8 * 4 * 64, 4, 64)), "strides")
    refused(lib, backward(size=16), "workspace too small")
    refused(lib, backward(ws=ctypes.c_void_p(4100)), "aligned")
    refused(lib, backward(dq=ctypes.c_void_p(4100)), "aligned")
    assert backward(batch=0) == 0
    assert lib.isa_block_attention_backward_workspace(attention(head_dim=7)) == 0
    assert lib.isa_block_attention_backward_workspace(attention()) >= 2 * 4 * 8 * 4


def test_attention_workspaces_stay_bounded(lib):
    """A launch's partial sums are those of some thousand blocks at most, whatever the sizes."""
    stride = {"q_strides": (0, 256, 64), "k_strides": (0, 128, 64), "v_strides": (0, 128, 64)}
    for sinks in (0, 4, 1000, 1 << 20):
        for window in (0, 1, 64, 5000):
            for kind in (0, 1):
                a = attention(type=kind, batch=1, queries=1 << 20, keys=1 << 20, window=window, sinks=sinks, **stride)
                planes = 3 * 4 * 4 * (1 << 20)
                assert planes <= lib.isa_block_attention_backward_workspace(a) <= planes + (400 << 20)
                assert lib.isa_block_attention_forward_workspace(a) == 0
            a = attention(batch=1, queries=1, keys=1 << 20, window=window, sinks=sinks, **stride)
            assert lib.isa_block_attention_forward_workspace(a) <= 1 << 20


def loss(**over):
    n = Loss(0, 4, 100, -100, 4096, 100, 4096)
    for k, v in over.items():
        setattr(n, k, v)
    return ctypes.byref(n)


def test_loss_refusals(lib):
    def with_grad(out=FAKE, grad=FAKE, ws=FAKE, size=1 << 30, **over):
        return lib.isa_block_loss_with_grad(loss(**over), 1.0, out, grad, 100, ws, size, None)

    refused(lib, lib.isa_block_loss_with_grad(None, 1.0, FAKE, FAKE, 1, FAKE, 0, None), "null")
    refused(lib, with_grad(type=-1), "type")
    refused(lib, with_grad(rows=-1), "rows")
    refused(lib, with_grad(rows=(1 << 24) + 1), "rows")
    refused(lib, with_grad(vocab=0), "vocab")
    refused(lib, with_grad(logits=None), "must be set")
    refused(lib, with_grad(targets=None), "must be set")
    refused(lib, with_grad(logits=4098), "aligned")
    refused(lib, with_grad(out=None), "must be set")
    refused(lib, with_grad(grad=None), "must be set")
    refused(lib, with_grad(grad=ctypes.c_void_p(4098)), "aligned")
    refused(lib, with_grad(size=0), "workspace too small")
    refused(lib, with_grad(ws=ctypes.c_void_p(4100)), "aligned")

    def forward(reduction=0, out=FAKE, size=1 << 30, **over):
        return lib.isa_block_loss_forward(loss(**over), reduction, out, None, None, FAKE, size, None)

    refused(lib, forward(reduction=3), "reduction")
    refused(lib, forward(out=None), "out is null")
    refused(lib, forward(size=0), "workspace too small")
    assert forward(reduction=2, rows=0) == 0

    def backward(reduction=0, stats=FAKE, count=FAKE, up=FAKE, grad=FAKE, **over):
        return lib.isa_block_loss_backward(loss(**over), reduction, stats, count, up, grad, 100, None)

    refused(lib, backward(reduction=-1), "reduction")
    refused(lib, backward(stats=None), "must be set")
    refused(lib, backward(count=None), "must be set")
    refused(lib, backward(up=None), "must be set")
    refused(lib, backward(grad=ctypes.c_void_p(4097)), "aligned")
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
