"""include/isa_train.h: what it declares the library exports, and bad arguments are refused before any HIP call (CPU only:
no kernel is launched here)."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

from isa.kernels.transformer_block import _hip
from tests.test_block_abi import F32, FAKE, I64, INT, SIZE, VP, Loss, Norm, refused

HEADER = Path(__file__).resolve().parents[1] / "include" / "isa_train.h"
ODD = ctypes.c_void_p(4097)


class Embedding(ctypes.Structure):
    _fields_ = [("type", INT), ("tokens", I64), ("dim", I64), ("vocab", I64), ("weight_stride", I64), ("ids", VP), ("weight", VP),
                ("scale", F32), ("places", I64), ("places_stride", I64), ("place_ids", VP), ("period", I64), ("place_weight", VP)]


class Dropout(ctypes.Structure):
    _fields_ = [("seed", VP), ("site", I64), ("threshold", INT)]


class Policy(ctypes.Structure):
    _fields_ = [("loss", Loss), ("old_logp", VP), ("advantages", VP), ("ref_logp", VP), ("low", F32), ("high", F32), ("kl", F32)]


class Preference(ctypes.Structure):
    _fields_ = [("loss", Loss), ("pairs", I64), ("tokens", I64), ("ref_logp", VP), ("beta", F32)]


EMB, DROP, POL, PREF, NORM, LOSS = (ctypes.POINTER(t) for t in (Embedding, Dropout, Policy, Preference, Norm, Loss))
SIGNATURES = {
    "isa_train_abi_version": (INT,),
    "isa_train_embedding_lists": (SIZE, EMB, INT, INT),
    "isa_train_embedding_forward": (INT, EMB, VP, INT, INT, I64, VP, SIZE, VP),
    "isa_train_embedding_backward_workspace": (SIZE, EMB, INT, INT),
    "isa_train_embedding_backward": (INT, EMB, VP, SIZE, VP, VP, VP, INT, INT, VP, SIZE, VP),
    "isa_train_dropout_apply": (INT, DROP, INT, I64, I64, VP, I64, VP, VP),
    "isa_train_dropout_norm_forward": (INT, NORM, DROP, VP, I64, VP, I64, VP, VP, VP, VP, VP),
    "isa_train_dropout_norm_backward": (INT, NORM, DROP, VP, VP, VP, I64, VP, VP, VP, VP, VP, VP, VP, SIZE, VP),
    "isa_train_policy_forward": (INT, POL, INT, VP, VP, VP, VP, VP, VP, SIZE, VP),
    "isa_train_policy_backward": (INT, LOSS, INT, VP, VP, VP, VP, VP, I64, VP),
    "isa_train_policy_with_grad": (INT, POL, F32, VP, VP, VP, I64, VP, SIZE, VP),
    "isa_train_preference_workspace": (SIZE, PREF),
    "isa_train_preference_forward": (INT, PREF, INT, VP, VP, VP, VP, VP, SIZE, VP),
    "isa_train_preference_backward": (INT, PREF, INT, VP, VP, VP, VP, I64, VP),
    "isa_train_preference_with_grad": (INT, PREF, F32, VP, VP, VP, I64, VP, SIZE, VP),
}


@pytest.fixture(scope="module", name="lib")
def _lib():
    lib = ctypes.CDLL(str(_hip.LIB_PATH))
    for name, (result, *arguments) in SIGNATURES.items():
        f = getattr(lib, name)
        f.restype, f.argtypes = result, arguments
    lib.isa_block_last_error.restype = ctypes.c_char_p
    return lib


def test_header_declares_what_the_library_exports(lib):
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    assert sorted(set(re.findall(r"\b(isa_train_\w+)\s*\(", text))) == sorted(SIGNATURES)
    version = int(re.search(r"#define ISA_TRAIN_ABI_VERSION (\d+)", text).group(1))
    assert lib.isa_train_abi_version() == version == _hip.load().TRAIN_ABI_VERSION


def changed(t, over):
    for k, v in over.items():
        setattr(t, k, v)
    return ctypes.byref(t)


def embedding(**over):
    return changed(Embedding(0, 6, 8, 10, 8, 4096, 4096, 1.0, 0, 0, None, 0, None), over)


def test_embedding_refusals(lib):
    def forward(y=FAKE, learn=0, learn_places=0, lists=None, size=0, **over):
        return lib.isa_train_embedding_forward(embedding(**over), y, learn, learn_places, -1, lists, size, None)

    refused(lib, lib.isa_train_embedding_forward(None, FAKE, 0, 0, -1, None, 0, None), "null")
    refused(lib, forward(type=3), "type")
    for name, bad in (("tokens", -1), ("tokens", (1 << 30) + 1), ("dim", 0), ("dim", (1 << 20) + 1), ("vocab", -1),
                      ("vocab", (1 << 24) + 1), ("places", -1), ("places", (1 << 24) + 1)):
        refused(lib, forward(**{name: bad}), "sizes out of range")
    refused(lib, forward(ids=None), "ids must be set")
    refused(lib, forward(y=None), "must be set")
    refused(lib, forward(weight=None), "must be set")
    refused(lib, forward(places=4, period=6), "place_weight must be set")
    refused(lib, forward(places=4, period=0, place_weight=4096), "period")
    refused(lib, forward(places=4, period=4, place_weight=4096), "period")
    refused(lib, forward(y=ODD), "aligned")
    refused(lib, forward(learn=1), "lists too small")
    refused(lib, forward(learn=1, lists=ctypes.c_void_p(4100), size=1 << 20), "lists must be")
    assert forward(tokens=0) == 0
    assert lib.isa_train_embedding_lists(embedding(type=9), 1, 1) == 0
    assert lib.isa_train_embedding_lists(embedding(), 1, 0) >= 4 * (6 + 11)
    # places that are counted need no list
    assert lib.isa_train_embedding_lists(embedding(places=4, period=6, place_weight=4096), 0, 1) == 0

    def backward(dy=FAKE, dw=FAKE, dp=None, lists=FAKE, size=1 << 20, listed=1, ws=None, ws_size=0, **over):
        return lib.isa_train_embedding_backward(embedding(**over), lists, size, dy, dw, dp, listed, 0, ws, ws_size, None)

    refused(lib, backward(listed=0), "no lists")
    refused(lib, backward(dp=FAKE), "no lists")
    refused(lib, backward(dy=None), "grad_y")
    refused(lib, backward(size=8), "lists too small")
    refused(lib, backward(dw=ODD), "aligned")
    refused(lib, backward(tokens=5000), "workspace too small")
    refused(lib, backward(tokens=5000, ws=ctypes.c_void_p(4100), ws_size=1 << 30), "workspace must be")
    assert backward(dw=None) == 0 and backward(vocab=0) == 0
    # tiles' sums stay bounded whatever the tokens
    for tokens in (1 << 12, 1 << 20, 1 << 30):
        assert lib.isa_train_embedding_backward_workspace(embedding(tokens=tokens), 1, 0) <= 2049 * (2 * 8 * 4 + 4) + 1024


def test_dropout_refusals(lib):
    def drop(**over):
        return changed(Dropout(4096, 0, 100), over)

    def apply(d=None, kind=0, rows=4, dim=8, x=FAKE, y=FAKE, **over):
        return lib.isa_train_dropout_apply(drop(**over), kind, rows, dim, x, dim, y, None)

    refused(lib, lib.isa_train_dropout_apply(None, 0, 1, 1, FAKE, 1, FAKE, None), "null")
    for bad in (-1, 65537):
        refused(lib, apply(threshold=bad), "threshold")
    refused(lib, apply(seed=None), "seed")
    refused(lib, apply(seed=4100), "seed")
    refused(lib, apply(kind=5), "type")
    refused(lib, apply(rows=-1), "rows")
    refused(lib, apply(dim=-1), "dim")
    refused(lib, apply(dim=(1 << 30) + 1), "dim")
    refused(lib, apply(rows=1 << 40, dim=1 << 30), "rows")
    refused(lib, apply(x=None), "must be set")
    refused(lib, apply(y=ODD), "aligned")
    assert apply(rows=0) == 0 and apply(dim=0) == 0

    def norm(**over):
        return changed(Norm(0, 0, 0, 4, 64, 1e-5, 4096, None), over)

    def forward(x=FAKE, h=FAKE, threshold=5, **over):
        return lib.isa_train_dropout_norm_forward(norm(**over), drop(threshold=threshold), x, 64, FAKE, 64, FAKE, h, None, None, None)

    refused(lib, forward(threshold=-2), "threshold")
    refused(lib, forward(x=None), "x must be set")
    refused(lib, forward(h=None), "go together")
    refused(lib, forward(dim=16385), "16384")
    assert forward(rows=0) == 0

    def backward(dx=FAKE, dw=FAKE, db=FAKE, ws=FAKE, size=1 << 30, **over):
        return lib.isa_train_dropout_norm_backward(norm(**over), drop(), FAKE, None, FAKE, 64, FAKE, FAKE, dx, FAKE, dw, db, ws, size, None)

    refused(lib, backward(dx=None), "grad_x must be set")
    refused(lib, backward(dw=None), "grad_weight")
    refused(lib, backward(size=16), "workspace too small")
    assert backward(rows=0, dw=None, db=None) == 0


def logits(rows, **over):
    t = Loss(0, rows, 100, -100, 4096, 100, 4096)
    for k, v in over.items():
        setattr(t, k, v)
    return t


def test_policy_refusals(lib):
    def policy(loss=None, **over):
        return changed(Policy(loss or logits(4), 4096, 4096, 4096, 0.8, 1.2, 0.1), over)

    def with_grad(out=FAKE, logp=FAKE, grad=FAKE, ws=FAKE, size=1 << 30, **over):
        return lib.isa_train_policy_with_grad(policy(**over), 1.0, out, logp, grad, 100, ws, size, None)

    def forward(reduction=0, out=FAKE, logp=FAKE, stats=None, slope=None, count=None, size=1 << 30, **over):
        return lib.isa_train_policy_forward(policy(**over), reduction, out, logp, stats, slope, count, FAKE, size, None)

    refused(lib, lib.isa_train_policy_with_grad(None, 1.0, FAKE, FAKE, FAKE, 1, FAKE, 0, None), "null")
    for call in (with_grad, forward):
        refused(lib, call(loss=logits(4, type=7)), "type")
        refused(lib, call(loss=logits(-1)), "rows")
        refused(lib, call(old_logp=None), "old_logp")
        refused(lib, call(advantages=None), "advantages")
        refused(lib, call(ref_logp=None), "kl needs")
        refused(lib, call(low=1.5), "bounds")
        refused(lib, call(low=-0.1), "bounds")
        refused(lib, call(high=float("nan")), "bounds")
        refused(lib, call(kl=-1.0), "kl must")
        refused(lib, call(out=None), "must be set")
        refused(lib, call(logp=None), "must be set")
        refused(lib, call(size=16), "workspace too small")
    refused(lib, with_grad(grad=None), "must be set")
    refused(lib, with_grad(grad=ODD), "aligned")
    refused(lib, with_grad(ws=ctypes.c_void_p(4100)), "aligned")
    refused(lib, forward(reduction=3), "reduction")
    refused(lib, forward(stats=FAKE), "go together")
    assert forward(reduction=2, loss=logits(0)) == 0

    def backward(reduction=0, stats=FAKE, slope=FAKE, count=FAKE, up=FAKE, grad=FAKE, **over):
        return lib.isa_train_policy_backward(ctypes.byref(logits(**{"rows": 4, **over})), reduction, stats, slope, count, up, grad, 100, None)

    refused(lib, backward(reduction=-1), "reduction")
    for name in ("stats", "slope", "count", "up", "grad"):
        refused(lib, backward(**{name: None}), "must be set")
    refused(lib, backward(grad=ODD), "aligned")
    assert backward(rows=0) == 0


def test_preference_refusals(lib):
    def preference(loss=None, **over):
        return changed(Preference(loss or logits(12), 2, 3, 4096, 0.1), over)

    def with_grad(out=FAKE, logp=FAKE, grad=FAKE, ws=FAKE, size=1 << 30, **over):
        return lib.isa_train_preference_with_grad(preference(**over), 1.0, out, logp, grad, 100, ws, size, None)

    def forward(reduction=0, out=FAKE, logp=FAKE, stats=None, slope=None, size=1 << 30, **over):
        return lib.isa_train_preference_forward(preference(**over), reduction, out, logp, stats, slope, FAKE, size, None)

    refused(lib, lib.isa_train_preference_with_grad(None, 1.0, FAKE, FAKE, FAKE, 1, FAKE, 0, None), "null")
    for call in (with_grad, forward):
        refused(lib, call(loss=logits(11)), "rows must be")
        refused(lib, call(pairs=-2, tokens=-3), "rows must be")
        refused(lib, call(pairs=1 << 40, loss=logits(0), tokens=0), "rows must be")
        refused(lib, call(ref_logp=None), "ref_logp")
        for beta in (0.0, -1.0, float("nan"), float("inf")):
            refused(lib, call(beta=beta), "beta")
        refused(lib, call(out=None), "must be set")
        refused(lib, call(logp=None), "must be set")
        refused(lib, call(size=16), "workspace too small")
    refused(lib, with_grad(grad=None), "must be set")
    refused(lib, with_grad(grad=ODD), "aligned")
    refused(lib, with_grad(ws=ctypes.c_void_p(4100)), "aligned")
    refused(lib, forward(reduction=5), "reduction")
    refused(lib, forward(stats=FAKE), "go together")
    assert forward(reduction=2, loss=logits(0), pairs=0, tokens=0) == 0
    assert lib.isa_train_preference_workspace(preference(loss=logits(11))) == 0

    def backward(reduction=0, stats=FAKE, slope=FAKE, up=FAKE, grad=FAKE, **over):
        return lib.isa_train_preference_backward(preference(**over), reduction, stats, slope, up, grad, 100, None)

    refused(lib, backward(reduction=3), "reduction")
    for name in ("stats", "slope", "up", "grad"):
        refused(lib, backward(**{name: None}), "must be set")
    refused(lib, backward(grad=ODD), "aligned")
    assert backward(loss=logits(0), pairs=0, tokens=0) == 0


def test_cpu_tensors_are_refused():
    from isa.kernels import transformer_block as ops

    x, w, t, f = torch.zeros(2, 8), torch.ones(8), torch.zeros(2, dtype=torch.int64), torch.zeros(2)
    seed, y = torch.zeros(2, dtype=torch.int64), torch.zeros(2, 1, 8)
    for call in (lambda: ops.embedding(t, x), lambda: ops.dropout(x, 0.5, seed),
                 lambda: ops.dropout_add_layer_norm(x, x, w, p=0.5, seed=seed), lambda: ops.policy_loss(x, t, f, f),
                 lambda: ops.policy_loss_with_grad(x, t, f, f), lambda: ops.preference_loss(y, t[:, None], f),
                 lambda: ops.preference_loss_with_grad(y, t[:, None], f)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_a_seeds_steps():
    from isa.operators.block import DropoutSeed

    s = DropoutSeed(key=-4)
    cpu = torch.device("cpu")
    assert s.step(3, cpu).tolist() == [-4, 0] and s.step(5, cpu).tolist() == [-4, 3] and s.state.tolist() == [-4, 8]
    with torch.inference_mode():
        made = DropoutSeed(key=1)
        assert made.step(1, cpu).tolist() == [1, 0]
    assert made.step(1, cpu).tolist() == [1, 1]
    torch.manual_seed(1)
    a = DropoutSeed().state
    torch.manual_seed(1)
    assert torch.equal(a, DropoutSeed().state) and not torch.equal(a, DropoutSeed().state)
