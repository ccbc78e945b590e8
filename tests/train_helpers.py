"""64-bit implementations of the training step's operators."""

from __future__ import annotations

import math

import torch

MASK = 0xFFFFFFFF


def philox(counter, key):
    """Philox4x32-10 of Python numbers: (four words) of four words and two."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & MASK, (a >> 32) ^ c[3] ^ k[1], a & MASK]
        k = [(k[0] + 0x9E3779B9) & MASK, (k[1] + 0xBB67AE85) & MASK]
    return c


def numbers(rows, dim, seed, site=0):
    """[rows, dim]: every element's 16-bit number, from Python's integers."""
    groups = -(-dim // 8)
    key, offset = seed[0] % 2 ** 64, (seed[1] + site) % 2 ** 64
    out = torch.empty(rows, groups * 8, dtype=torch.int64)
    for g in range(rows * groups):
        words = philox((g & MASK, g >> 32, offset & MASK, offset >> 32), (key & MASK, key >> 32))
        out.view(-1)[8 * g: 8 * g + 8] = torch.tensor([(w >> s) & 0xFFFF for w in words for s in (0, 16)])
    return out[:, :dim]


def factors(rows, dim, p, seed, site=0):
    """[rows, dim] in 64 bits: what dropout multiplies an element by."""
    least = round(65536 * p)
    if least == 65536:
        return torch.zeros(rows, dim, dtype=torch.float64)
    return (numbers(rows, dim, seed, site) >= least).double() * (65536.0 / (65536 - least))


def embedding64(ids, weight, scale, positions=None, position_weight=None, padding=None, dy=None):
    """(y, dweight, dposition_weight) by the formulas, on the CPU; ids and positions [tokens]."""
    w, ids = weight.detach().double().cpu(), ids.cpu().long()
    inside = (ids >= 0) & (ids < w.shape[0])
    y = scale * w[ids.where(inside, torch.zeros_like(ids))] if w.shape[0] else torch.zeros(len(ids), w.shape[1]).double()
    y = y.masked_fill(~inside[:, None], math.nan)
    there = None
    if position_weight is not None:
        p, at = position_weight.detach().double().cpu(), positions.cpu().long()
        there = (at >= 0) & (at < p.shape[0])
        y = (y + p[at.where(there, torch.zeros_like(at))]).masked_fill(~there[:, None], math.nan)
    if dy is None:
        return y, None, None
    g = dy.detach().double().cpu().reshape(len(ids), -1)
    if padding is not None:
        inside = inside & (ids != padding)
    dw = torch.zeros_like(w).index_add_(0, ids[inside], scale * g[inside])
    dp = None if there is None else torch.zeros_like(p).index_add_(0, at[there], g[there])
    return y, dw, dp


def logp64(x, targets, ignore):
    """(l of each row, 0 where ignored; softmax; one-hot; which rows count)."""
    x, t = x.detach().double().cpu(), targets.cpu()
    counted = t != ignore
    at = t.masked_fill(~counted, 0)[:, None]
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    l = (x.gather(1, at) - top - torch.log(total))[:, 0]
    hot = torch.zeros_like(x).scatter_(1, at, 1.0)
    return l.masked_fill(~counted, 0.0), e / total, hot, counted


def policy64(x, actions, old, advantages, ref, low, high, kl, ignore):
    """(losses of rows, gradients of each row's own loss, l) of [rows, vocab]."""
    l, p, hot, counted = logp64(x, actions, ignore)
    a, r = advantages.double().cpu(), torch.exp(l - old.double().cpu())
    held = r.clamp(1.0 - low, 1.0 + high)
    loss = -torch.minimum(r * a, held * a)
    slope = torch.where(r * a <= held * a, -r * a, torch.zeros_like(a))
    if kl:
        gap = ref.double().cpu() - l
        loss = loss + kl * (torch.expm1(gap) - gap)
        slope = slope - kl * torch.expm1(gap)
    loss, slope = loss.masked_fill(~counted, 0.0), slope.masked_fill(~counted, 0.0)
    return loss, slope[:, None] * (hot - p), l


def preference64(x, targets, ref, beta, ignore):
    """(losses of pairs, gradients [2 pairs, tokens, vocab] of each pair's own loss, L)."""
    b, n, v = x.shape
    l, p, hot, counted = logp64(x.reshape(b * n, v), targets.reshape(-1), ignore)
    total = l.view(b, n).sum(1)
    over = total - ref.double().cpu()
    m = beta * (over[: b // 2] - over[b // 2:])
    loss = torch.nn.functional.softplus(-m)
    slope = torch.cat([-beta * torch.sigmoid(-m), beta * torch.sigmoid(-m)]).repeat_interleave(n) * counted
    return loss, (slope[:, None] * (hot - p)).view(b, n, v), total
