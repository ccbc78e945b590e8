"""What the training step's operators do not take they refuse, and what stands for other memory they read as it is."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu


def calls(dev):
    """(name, function of floating tensors, those tensors, whether autograd follows it)."""
    from isa.kernels import transformer_block as ops

    g = torch.Generator(device=dev).manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    ids = torch.tensor([[1, 2, 3], [0, 1, 1]], device=dev)
    t = torch.tensor([1, 2, 3, 0], device=dev)
    t2 = t.view(2, 2)
    seed = torch.tensor([5, 6], device=dev)
    old, a, ref = rnd(4) - 3.0, rnd(4), rnd(4) - 3.0
    ref2 = ref[:2].clone()
    return [("embedding", lambda w, p: ops.embedding(ids, w, position_weight=p, scale=2.0), [rnd(5, 16), rnd(3, 16)], True),
            ("dropout", lambda x: ops.dropout(x, 0.5, seed), [rnd(4, 32)], True),
            ("dropout_add_layer_norm", lambda x, r, w, b: ops.dropout_add_layer_norm(x, r, w, b, p=0.5, seed=seed)[0],
             [rnd(4, 32), rnd(4, 32), rnd(32), rnd(32)], True),
            ("policy_loss", lambda x: ops.policy_loss(x, t, old, a, ref_logp=ref, kl=0.1)[0], [rnd(4, 10)], True),
            ("preference_loss", lambda x: ops.preference_loss(x, t2, ref2)[0], [rnd(2, 2, 10)], True),
            ("policy_loss_with_grad", lambda x: ops.policy_loss_with_grad(x, t, old, a)[0], [rnd(4, 10)], False),
            ("preference_loss_with_grad", lambda x: ops.preference_loss_with_grad(x, t2, ref2)[0],
             [rnd(2, 2, 10)], False)]


@pytest.mark.parametrize("grad", [False, True], ids=["direct", "tracked"])
def test_forward_mode_is_refused(cuda_device, grad):
    for name, f, args, _ in calls(cuda_device):
        for i in range(len(args)):
            print(f"[case] tangent of argument {i} of {name}", flush=True)
            with fwAD.dual_level():
                dual = [a.clone().requires_grad_(grad) for a in args]
                dual[i] = fwAD.make_dual(dual[i], torch.ones_like(args[i]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f(*dual)
                with fwAD._set_fwd_grad_enabled(False):
                    assert torch.equal(f(*dual), f(*args))


def test_forward_mode_of_what_is_held_fixed_is_refused(cuda_device):
    from isa.kernels.transformer_block import policy_loss, preference_loss

    x, t = torch.randn(4, 10, device=cuda_device), torch.tensor([1, 2, 3, 0], device=cuda_device)
    f = torch.zeros(4, device=cuda_device)
    with fwAD.dual_level():
        d = fwAD.make_dual(f, torch.ones_like(f))
        for args in ((d, f, f), (f, d, f), (f, f, d)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                policy_loss(x, t, args[0], args[1], ref_logp=args[2], kl=0.1)
        with pytest.raises(RuntimeError, match="forward-mode"):
            preference_loss(x.view(2, 2, 10), t.view(2, 2), fwAD.make_dual(f[:2].clone(), torch.ones(2, device=cuda_device)))


def test_backward_refusals(cuda_device):
    from torch.fx.experimental.proxy_tensor import make_fx

    for name, f, args, follows in calls(cuda_device):
        if not follows:
            continue
        print(f"[case] {name}'s gradient", flush=True)
        leaves = [a.clone().requires_grad_(True) for a in args]
        out = f(*leaves)
        with pytest.raises(RuntimeError, match="first derivatives only"):
            torch.autograd.grad(out.sum(), leaves, create_graph=True)
        out = f(*leaves)
        with fwAD.dual_level():
            up = fwAD.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, leaves, up, retain_graph=True)
        out = f(*leaves)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(lambda g: torch.autograd.grad(out, leaves, g))(torch.ones_like(out))
        # twice through one graph gives the same bits
        out = f(*leaves)
        one = torch.autograd.grad(out, leaves, torch.ones_like(out), retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(one, torch.autograd.grad(out, leaves, torch.ones_like(out))))


@pytest.mark.parametrize("grad", [False, True], ids=["direct", "tracked"])
def test_traces_are_refused(cuda_device, grad):
    from torch.fx.experimental.proxy_tensor import make_fx

    for name, f, args, _ in calls(cuda_device):
        print(f"[case] trace of {name}", flush=True)
        args = [a.requires_grad_(grad) for a in args]
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, tuple(args), check_trace=False)
        for mode in ("real", "fake"):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                make_fx(f, tracing_mode=mode)(*args)
        assert torch.isfinite(f(*args)).all()


def negative_view(t):
    """-t, as a view of t's own elements."""
    return torch.view_as_complex(torch.stack([torch.zeros_like(t), t], -1)).conj().imag


def test_negative_views(cuda_device):
    for make in (negative_view, torch._neg_view):
        for name, f, args, follows in calls(cuda_device):
            print(f"[case] {make.__name__} of {name}'s operands", flush=True)
            views = [make(a).detach().requires_grad_(True) for a in args]
            copies = [(-a).requires_grad_(True) for a in args]
            assert views[0].is_neg()
            a, b = f(*views), f(*copies)
            torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)
            if follows:
                up = torch.randn_like(b)
                want = torch.autograd.grad(b, copies, -up)
                for x, y in zip(torch.autograd.grad(a, views, make(up)), want):
                    torch.testing.assert_close(x, y, rtol=1e-5, atol=1e-5)
    from isa.kernels.transformer_block import dropout, embedding, policy_loss_with_grad

    # integers and what is held fixed
    t, f = torch.tensor([1, 2, 3, 0], device=cuda_device), torch.randn(4, device=cuda_device)
    x = torch.randn(4, 16, device=cuda_device)
    assert torch.equal(embedding(torch._neg_view(-t), x), embedding(t, x))
    assert torch.equal(dropout(x, 0.5, torch._neg_view(torch.tensor([-3, -4], device=cuda_device))),
                       dropout(x, 0.5, torch.tensor([3, 4], device=cuda_device)))
    a = policy_loss_with_grad(x, t, torch._neg_view(-f), torch._neg_view(-f))
    assert all(torch.equal(p, q) for p, q in zip(a, policy_loss_with_grad(x, t, f, f)))


def test_arguments_that_do_not_fit(cuda_device):
    from isa.kernels import transformer_block as ops

    dev = cuda_device
    w, ids = torch.randn(5, 8, device=dev), torch.tensor([[1, 2], [3, 4]], device=dev)
    seed = torch.tensor([1, 2], device=dev)
    x, one = torch.randn(4, 8, device=dev), torch.ones(8, device=dev)
    t, f = torch.tensor([1, 2, 3, 0], device=dev), torch.zeros(4, device=dev)
    y, u = torch.randn(4, 3, 8, device=dev), torch.zeros(4, 3, dtype=torch.int64, device=dev)
    leaf = torch.zeros(4, device=dev, requires_grad=True)

    def refused(match, f, *a, **k):
        with pytest.raises(RuntimeError, match=match):
            f(*a, **k)

    refused("must be int64 or int32", ops.embedding, ids.float(), w)
    refused("must be on", ops.embedding, ids.cpu(), w)
    refused(r"must be \[rows, dim\]", ops.embedding, ids, w[0])
    refused(r"must be \[rows, dim\]", ops.embedding, ids, w[:, :0])
    refused("weight must be float32", ops.embedding, ids, w.double())
    refused("scale must be finite", ops.embedding, ids, w, scale=float("nan"))
    refused("padding_index", ops.embedding, ids, w, padding_index=5)
    refused("padding_index", ops.embedding, ids, w, padding_index=-1)
    refused("positions need position_weight", ops.embedding, ids, w, positions=ids)
    refused("must broadcast", ops.embedding, ids, w, positions=ids.view(-1), position_weight=w)
    refused("must be int64 or int32", ops.embedding, ids, w, positions=ids.double(), position_weight=w)
    refused("as weight is", ops.embedding, ids, w, position_weight=w.half())
    refused("as weight is", ops.embedding, ids, w, position_weight=w[:, :4])
    refused(r"must be \[rows, dim\] of 1", ops.embedding, ids, w, positions=ids, position_weight=w[:0])
    refused("do not fit a table of 1 positions", ops.embedding, ids, w, position_weight=w[:1])
    for p in (-0.1, 1.1, float("nan")):
        refused("p must be 0 to 1", ops.dropout, x, p, seed)
    refused("seed must be int64", ops.dropout, x, 0.5, seed.int())
    refused("seed must be int64", ops.dropout, x, 0.5, seed[:1])
    refused("seed must be on", ops.dropout, x, 0.5, seed.cpu())
    refused("x must be float32", ops.dropout, x.double(), 0.5, seed)
    refused("x must be", ops.dropout, x[0, 0], 0.5, seed)
    refused("one shape", ops.dropout_add_layer_norm, x[:2], x, one, p=0.5, seed=seed)
    refused("p must be 0 to 1", ops.dropout_add_layer_norm, x, x, one, p=2.0, seed=seed)
    refused("seed must be", ops.dropout_add_layer_norm, x, x, one, p=0.5, seed=seed.float())
    for loss in (ops.policy_loss, ops.policy_loss_with_grad):
        refused("actions must be int64", loss, x, t.int(), f, f)
        refused("actions must be int64", loss, x, t[:3], f, f)
        refused("old_logp must be torch.float32", loss, x, t, f.half(), f)
        refused("advantages must be torch.float32", loss, x, t, f, f[:3])
        refused("ref_logp must be torch.float32", loss, x, t, f, f, ref_logp=f[:1], kl=0.1)
        refused("kl needs ref_logp", loss, x, t, f, f, kl=0.1)
        refused("kl must be finite", loss, x, t, f, f, kl=-0.1, ref_logp=f)
        refused("kl must be finite", loss, x, t, f, f, kl=float("inf"), ref_logp=f)
        refused("clip must be", loss, x, t, f, f, clip=1.5)
        refused("clip must be", loss, x, t, f, f, clip=(0.1, -0.1))
        refused("must be on", loss, x, t, f.cpu(), f)
    refused("detach it", ops.policy_loss, x, t, leaf, f)
    refused("detach it", ops.policy_loss, x, t, f, leaf)
    refused("reduction must be", ops.policy_loss, x, t, f, f, reduction="max")
    for loss in (ops.preference_loss, ops.preference_loss_with_grad):
        refused("chosen sequences first", loss, y[:3], u[:3], f[:3])
        refused("chosen sequences first", loss, x, t, f)
        refused("targets must be int64", loss, y, u[:2], f)
        refused("ref_logp must be torch.float32", loss, y, u, f[:2])
        for beta in (0.0, -1.0, float("nan"), float("inf"), 1e-60):
            refused("beta must be positive", loss, y, u, f, beta=beta)
    refused("detach it", ops.preference_loss, y, u, leaf)
    refused("reduction must be", ops.preference_loss, y, u, f, reduction="max")
