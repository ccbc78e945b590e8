"""64-bit implementations of the block's operators and the error measure of their tests."""

from __future__ import annotations

import math

import torch

# unit roundoffs: half the distance from 1 to the next number
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def off(got: torch.Tensor, want: torch.Tensor):
    """(2-norm of the difference over the 2-norm of `want`, largest difference over the largest value)."""
    assert got.shape == want.shape, (got.shape, want.shape)
    g, w = got.detach().double().cpu(), want.detach().double().cpu()
    assert torch.isfinite(g).all()
    if not w.numel():
        return 0.0, 0.0
    d, n, top = (g - w), float(w.norm()), float(w.abs().max())
    if n == 0.0:
        return (0.0, 0.0) if float(d.abs().max()) == 0.0 else (math.inf, math.inf)
    return float(d.norm()) / n, float(d.abs().max()) / top


def close(got, want, tol, what=""):
    """The 2-norm's error within tol, no single one past eight times that of the largest value."""
    rel, big = off(got, want)
    print(f"  {what}: {rel:.2e} (largest {big:.2e}), tolerance {tol:.2e}", flush=True)
    assert rel <= tol and big <= 8 * tol, (what, rel, big, tol)


def layer_norm64(h, weight, bias, eps, dy=None, dh=None):
    """(y, dh, dw, db) by the formulas."""
    h, w = h.double(), weight.double()
    c = h - h.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(c.square().mean(-1, keepdim=True) + eps)
    n = c * rstd
    y = n * w + (0.0 if bias is None else bias.double())
    if dy is None:
        return (y,)
    dy = dy.double()
    dn = dy * w
    g = rstd * (dn - dn.mean(-1, keepdim=True) - n * (dn * n).mean(-1, keepdim=True))
    if dh is not None:
        g = g + dh.double()
    lead = tuple(range(dy.dim() - 1))
    return y, g, (dy * n).sum(lead), dy.sum(lead)


def visible(batch, queries, keys, window, sinks, lengths):
    n = torch.as_tensor(lengths if lengths is not None else [keys] * batch).clamp(0, keys).view(-1, 1, 1)
    p = n - queries + torch.arange(queries).view(1, -1, 1)
    j = torch.arange(keys).view(1, 1, -1)
    seen = (j <= p) & (p >= 0)
    return seen if window is None else seen & ((j < sinks) | (p - j < window))


def attention64(q, k, v, window, sinks, scale, lengths, dout=None):
    """(out, dq, dk, dv) by the formulas, on the CPU; what a query does not see has no part in it."""
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    b, m, h, d = q.shape
    n, kv = k.shape[1], k.shape[2]
    seen = visible(b, m, n, window, sinks, None if lengths is None else [int(x) for x in lengths])
    any_sees = seen.any(1)[:, :, None, None]
    k, v = (torch.where(any_sees, t, torch.zeros_like(t)) for t in (k, v))
    kh, vh = (t.repeat_interleave(h // kv, 2).permute(0, 2, 1, 3) for t in (k, v))
    qh = q.permute(0, 2, 1, 3)
    s = (qh @ kh.transpose(2, 3)) * scale
    s = s.masked_fill(~seen[:, None], -math.inf)
    top = s.amax(-1, keepdim=True) if n else s.sum(-1, keepdim=True)
    e = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
    total = e.sum(-1, keepdim=True)
    p = e / total.masked_fill(total == 0.0, 1.0)
    out = p @ vh
    back = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731
    if dout is None:
        return (back(out),)
    g = back(dout.detach().double().cpu())
    dv = p.transpose(2, 3) @ g
    dp = g @ vh.transpose(2, 3)
    ds = p * (dp - (dp * p).sum(-1, keepdim=True)) * scale
    dq, dk = ds @ kh, ds.transpose(2, 3) @ qh
    shared = lambda t: back(t).reshape(b, n, kv, h // kv, d).sum(3)  # noqa: E731
    return back(out), back(dq), shared(dk), shared(dv)


def cross_entropy64(x, targets, ignore):
    """(losses of rows, gradients of each row's own loss) of [rows, vocab]."""
    x = x.detach().double().cpu()
    t = targets.cpu()
    counted = t != ignore
    at = t.masked_fill(~counted, 0)[:, None]
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    loss = (torch.log(total) + top - x.gather(1, at))[:, 0]
    grad = (e / total).scatter_add(1, at, torch.full_like(total, -1.0))
    return loss * counted, grad * counted[:, None]
