"""What the block's operators do not give they refuse: forward-mode derivatives, whose tangent would be missing
without a word, and traces, which would hold an allocation and not what fills it."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu


def calls(dev):
    """(name, function of floating tensors, those tensors)."""
    from isa.kernels.transformer_block import (add_layer_norm, cross_entropy, cross_entropy_with_grad, layer_norm,
                                               window_attention)

    g = torch.Generator(device=dev).manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    t = torch.tensor([1, 2, 3, 0], device=dev)
    return [("layer_norm", lambda x, w, b: layer_norm(x, w, b), [rnd(4, 32), rnd(32), rnd(32)]),
            ("add_layer_norm", lambda x, r, w, b: add_layer_norm(x, r, w, b)[0], [rnd(4, 32), rnd(4, 32), rnd(32), rnd(32)]),
            ("window_attention", lambda q, k, v: window_attention(q, k, v),
             [rnd(1, 4, 2, 16), rnd(1, 4, 2, 16), rnd(1, 4, 2, 16)]),
            ("cross_entropy", lambda x: cross_entropy(x, t), [rnd(4, 10)]),
            ("cross_entropy_with_grad", lambda x: cross_entropy_with_grad(x, t)[0], [rnd(4, 10)])]


@pytest.mark.parametrize("grad", [False, True], ids=["direct", "tracked"])
def test_forward_mode_is_refused(cuda_device, grad):
    for name, f, args in calls(cuda_device):
        for i in range(len(args)):
            print(f"[case] tangent of argument {i} of {name}", flush=True)
            with fwAD.dual_level():
                dual = [a.clone().requires_grad_(grad) for a in args]
                dual[i] = fwAD.make_dual(dual[i], torch.ones_like(args[i]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f(*dual)
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                    f(*dual)
                # a tangent that is not followed is not in the way
                with fwAD._set_fwd_grad_enabled(False):
                    assert torch.equal(f(*dual), f(*args))
        assert torch.equal(f(*args), f(*args))


def test_forward_mode_through_the_backward_is_refused(cuda_device):
    """A gradient that comes with a tangent (the backward pass is linear in it) would lose it."""
    for name, f, args in calls(cuda_device)[:4]:
        print(f"[case] tangent of {name}'s gradient", flush=True)
        leaves = [a.clone().requires_grad_(True) for a in args]
        with fwAD.dual_level():
            out = f(*leaves)
            up = fwAD.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, leaves, up)


@pytest.mark.parametrize("grad", [False, True], ids=["direct", "tracked"])
def test_traces_are_refused(cuda_device, grad):
    from torch.fx.experimental.proxy_tensor import make_fx

    for name, f, args in calls(cuda_device):
        print(f"[case] trace of {name}", flush=True)
        args = [a.requires_grad_(grad) for a in args]
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, tuple(args), check_trace=False)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(f)(*args)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(f, tracing_mode="fake")(*args)
        assert torch.isfinite(f(*args)).all()


def test_traces_of_the_backward_are_refused(cuda_device):
    from torch.fx.experimental.proxy_tensor import make_fx

    for name, f, args in calls(cuda_device)[:4]:
        print(f"[case] trace of {name}'s gradient", flush=True)
        leaves = [a.requires_grad_(True) for a in args]
        out = f(*leaves)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(lambda g: torch.autograd.grad(out, leaves, g))(torch.ones_like(out))
