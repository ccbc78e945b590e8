"""fp16 gradients of attention keep their precision where rows' gradients differ by many powers of two: each
key's and each query's own size decides how its ds is scaled.

Tolerances (2-norm of the error of a key's or query's gradients, u = 2^-11): ds and the result are rounded
once each, uniformly spread errors of at most u, some 0.4 u in the mean: sqrt(2) 0.4 u, and with p rounded too
for dv; 2 u covers that. What is below fp16's smallest number adds 2^-25 an element.
"""

from __future__ import annotations

import math

import pytest
import torch

from tests.block_helpers import UNIT, attention64, off

pytestmark = pytest.mark.gpu

U = UNIT[torch.float16]


def inputs(dev, b, m, n, h, kv, d, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(*shape, generator=g, device=dev).half()
            for shape in ((b, m, h, d), (b, n, kv, d), (b, n, kv, d), (b, m, h, d))]


def parts_close(got, want, parts, what):
    for name, at in parts:
        w = want[at]
        tol = 2 * U + 2.0 ** -25 * math.sqrt(w.numel()) / float(w.norm())
        rel, _ = off(got[at], w)
        print(f"  {what}, {name}: {rel:.2e}, tolerance {tol:.2e}", flush=True)
        assert rel <= tol, (what, name, rel, tol)


@pytest.mark.parametrize("ratio", [2.0 ** 10, 2.0 ** 14, 2.0 ** 18])
@pytest.mark.parametrize("size", [(1, 200, 2, 1, 64), (1, 900, 2, 2, 128), (2, 300, 4, 2, 32)], ids=str)
def test_one_row_of_large_gradients(cuda_device, size, ratio):
    """The keys that the row does not see, and the other queries, are as exact as without it."""
    from isa.kernels.transformer_block import window_attention

    b, n, h, kv, d = size
    print(f"[case] one row's gradient {ratio} times the others', {size}", flush=True)
    q, k, v, g = inputs(cuda_device, b, n, n, h, kv, d, seed=n + d)
    row = n // 3
    g = (g.float() * 2.0 ** -6).half()
    g[0, row] = (g[0, row].float() * ratio * 2.0 ** -4).clamp(-60000, 60000).half()
    want = attention64(q, k, v, 40, 2, 1.0 / math.sqrt(d), None, g)
    seeing = [t.requires_grad_(True) for t in (q, k, v)]
    out = window_attention(*seeing, window=40, sinks=2)
    dq, dk, dv = torch.autograd.grad(out, seeing, g)
    parts = [("keys behind the row", (0, slice(row + 1, None))), ("keys it sees", (0, slice(row - 39, row + 1))),
             ("keys before its window", (0, slice(2, row - 39)))]
    if b > 1:
        parts.append(("the other sequence", (1,)))
    parts_close(dk, want[2], parts, "dk")
    parts_close(dv, want[3], parts[:1] + parts[2:], "dv")
    parts_close(dq, want[1], [("the row", (0, row)), ("rows before", (0, slice(1, row))), ("rows behind", (0, slice(row + 1, None)))],
                "dq")
    leaves = [k.detach().clone().requires_grad_(True), v.detach().clone().requires_grad_(True)]
    out = window_attention(q.detach(), *leaves, window=40, sinks=2)
    parts_close(torch.autograd.grad(out, leaves, g)[0], want[2], parts, "dk alone")


def test_large_values(cuda_device):
    """Values of some 1000, aligned with the gradients: ds of gradients scaled to one would pass fp16's range."""
    from isa.kernels.transformer_block import window_attention

    print("[case] large values", flush=True)
    q, k, v, g = inputs(cuda_device, 1, 150, 150, 2, 2, 128, seed=2)
    side = torch.where(torch.arange(150, device=cuda_device) % 2 == 0, 1500.0, -1500.0)[None, :, None, None]
    v, g = (side + v.float()).half(), ((1.0 + 0.1 * g.float()) * 2.0 ** -10).half()
    want = attention64(q, k, v, None, 0, 1.0 / math.sqrt(128), None, g)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(window_attention(*leaves), leaves, g)
    for x, w, name in zip(grads, want[1:], ("dq", "dk", "dv")):
        assert torch.isfinite(x).all(), name
        parts_close(x[0], w[0], [("all", slice(1, None))], name)
