"""Views that stand for the negative of their memory (the imaginary part of a conjugate) give what their
copies give, as operands and as gradients."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def negative_view(t):
    """-t, as a view of t's own elements."""
    assert not t.is_neg()
    n = torch.view_as_complex(torch.stack([torch.zeros_like(t), t], -1)).conj().imag
    assert n.is_neg() and torch.equal(n, -t)
    return n


def test_negative_views(cuda_device):
    from isa.kernels.transformer_block import (add_layer_norm, cross_entropy, cross_entropy_with_grad, layer_norm,
                                               window_attention)

    g = torch.Generator(device=cuda_device).manual_seed(0)
    rnd = lambda *s: torch.randn(s, generator=g, device=cuda_device)  # noqa: E731
    t = torch.tensor([1, 2, 3, 0], device=cuda_device)
    # contiguous ones too, which contiguous() leaves as they are
    makers = (negative_view, torch._neg_view)
    for make in makers:
        for name, f, args in (("layer_norm", lambda x, w, b: layer_norm(x, w, b), [rnd(4, 32), rnd(32), rnd(32)]),
                              ("add_layer_norm", lambda *a: add_layer_norm(*a)[0], [rnd(4, 32), rnd(4, 32), rnd(32), rnd(32)]),
                              ("window_attention", lambda *a: window_attention(*a), [rnd(1, 4, 2, 16) for _ in range(3)]),
                              ("cross_entropy", lambda x: cross_entropy(x, t), [rnd(4, 10)])):
            print(f"[case] {make.__name__} of {name}'s operands", flush=True)
            views = [make(a).detach().requires_grad_(True) for a in args]
            copies = [(-a).requires_grad_(True) for a in args]
            a, b = f(*views), f(*copies)
            torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)
            up = rnd(*a.shape)
            want = torch.autograd.grad(b, copies, -up, retain_graph=True)
            for x, y in zip(torch.autograd.grad(a, views, make(up)), want):
                torch.testing.assert_close(x, y, rtol=1e-5, atol=1e-5)
            with torch.no_grad():
                torch.testing.assert_close(f(*views), b, rtol=1e-5, atol=1e-5)
        x = rnd(4, 10)
        torch.testing.assert_close(cross_entropy_with_grad(make(x), t), cross_entropy_with_grad(-x, t), rtol=1e-5, atol=1e-5)
