"""The public operators of a transformer block around its FFN, with their gradients."""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from isa.kernels.transformer_block import _hip, ops


class _LayerNormFn(torch.autograd.Function):
    """x None: y of residual; else (y, h)."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        ctx.set_materialize_grads(False)
        shape = residual.shape
        r2 = ops.rows_of(residual)
        x2 = None if x is None else ops.rows_of(x)
        weight = weight.contiguous()
        y, h, stats = ops.norm_forward(x2, r2, weight, None if bias is None else bias.contiguous(), eps, True)
        ctx.x_dtype = residual.dtype if x is None else x.dtype
        if x is None:
            ctx.save_for_backward(residual, weight, stats)
            return y.view(shape)
        h = h.view(shape)
        ctx.save_for_backward(h, weight, stats)
        return y.view(shape), h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, stats = ctx.saved_tensors
        need_x, need_r, need_w, need_b = ctx.needs_input_grad[:4]
        shape = h.shape
        if dy is None:  # only h was used
            dy = torch.zeros_like(h)
        h2 = ops.rows_of(h)
        dx, dr, dw, db = ops.norm_backward(ops.rows_of(dy), None if dh is None else ops.rows_of(dh), h2, stats,
                                           weight, ctx.x_dtype, need_w, need_b)
        dr = dr.view(shape)
        dx = dr if dx is None else dx.view(shape)
        return dx if need_x else None, dr if need_r else None, dw if need_w else None, db if need_b else None, None


def _tracked(*tensors: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension (at most 16384
    elements), in x's type, with statistics in fp32.

    x: float32, bfloat16 or float16; weight and bias: x's type or float32."""
    ops.check_norm(None, x, weight, bias)
    if _tracked(x, weight, bias):
        return _LayerNormFn.apply(None, x, weight, bias, float(eps))
    y, _, _ = ops.norm_forward(None, ops.rows_of(x), weight.contiguous(),
                               None if bias is None else bias.contiguous(), float(eps), False)
    return y.view(x.shape)


def add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                   bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, h): h = x + residual, rounded to residual's type, and y = layer_norm(h, weight, bias, eps).

    x is a branch's output, residual the stream it joins: of one type, or a 16-bit x beside a
    float32 residual (autocast). One pass forward and one backward, which takes the gradient
    that reaches h past the norm along."""
    ops.check_norm(x, residual, weight, bias)
    if _tracked(x, residual, weight, bias):
        return _LayerNormFn.apply(x, residual, weight, bias, float(eps))
    y, h, _ = ops.norm_forward(ops.rows_of(x), ops.rows_of(residual), weight.contiguous(),
                               None if bias is None else bias.contiguous(), float(eps), False)
    return y.view(residual.shape), h.view(residual.shape)


class _WindowAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, scale, key_lengths):
        q, k, v = (ops.attention_operand(t) for t in (q, k, v))
        out, rest, lse = ops.attention_forward(q, k, v, window, sinks, scale, key_lengths, True)
        ctx.save_for_backward(q, k, v, out, rest, lse, key_lengths)
        ctx.how = (window, sinks, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, rest, lse, key_lengths = ctx.saved_tensors
        need_q, need_k, need_v = ctx.needs_input_grad[:3]
        dq, dk, dv = ops.attention_backward(q, k, v, out, rest, lse, dout, *ctx.how, key_lengths, need_q,
                                            need_k or need_v)
        return dq, dk if need_k else None, dv if need_v else None, None, None, None, None


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: Optional[int] = None,
                     sinks: int = 0, scale: Optional[float] = None,
                     key_lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention over the last `window` tokens (None: over all) and the first `sinks` ones.

    q: [batch, queries, heads, head_dim]; k, v: [batch, keys, kv_heads, head_dim], all float32,
    bfloat16 or float16, in any strides (views of a joint projection or a longer cache are read in
    place where a head's elements are adjacent and 16-byte aligned). heads is a multiple of
    kv_heads: query heads in order share a key head. head_dim: a multiple of 8 up to 128.

    The queries are the last tokens of their sequence, which is key_lengths[b] keys long (int32 or
    int64 [batch] on the device; None: all keys; values are held to 0 .. keys). The query at position
    p sees key j iff j <= p and (j < sinks or p - j < window). So one call takes a whole prompt
    (queries == keys), a chunk of it or a single token over a cache. What lies behind a sequence's
    end is not read. A query that sees no key (more queries than keys) gives zeros and takes no
    gradient.

    Softmax and sums are fp32; scale is 1 / sqrt(head_dim) unless given. In 16-bit types the weights
    p, and in the backward p and ds, are rounded to that type for the matrix cores. Of a key that some
    but not all queries of a tile see, an infinity or NaN in v reaches the others too."""
    ops.check_attention(q, k, v, window, sinks, scale, key_lengths)
    scale = 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale)
    if key_lengths is not None:
        key_lengths = key_lengths.to(torch.int32).contiguous()
    if _tracked(q, k, v):
        return _WindowAttentionFn.apply(q, k, v, window, int(sinks), scale, key_lengths)
    q, k, v = (ops.attention_operand(t) for t in (q, k, v))
    return ops.attention_forward(q, k, v, window, int(sinks), scale, key_lengths, False)[0]


def _loss_operands(logits: torch.Tensor, targets: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    return ops.rows_of(logits), targets.reshape(-1).contiguous()


class _CrossEntropyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, ignore_index, reduction):
        x, t = _loss_operands(logits, targets)
        loss, stats, count = ops.loss_forward(x, t, ignore_index, reduction, True)
        ctx.save_for_backward(x, t, stats, count)
        ctx.how = (ignore_index, reduction)
        ctx.shape = logits.shape
        return loss.view(targets.shape) if reduction == "none" else loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        x, t, stats, count = ctx.saved_tensors
        grad = ops.loss_backward(x, t, *ctx.how, stats, count, dloss)
        return grad.view(ctx.shape) if grad.is_contiguous() else grad.reshape(ctx.shape), None, None, None


def cross_entropy(logits: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
                  reduction: str = "mean") -> torch.Tensor:
    """-log softmax(logits)[target] over the last dimension, as float32.

    logits: [..., vocab], float32, bfloat16 or float16; targets: int64 [...]. Rows whose target is
    ignore_index count nowhere; reduction is "mean" (over the others), "sum" or "none". Any other
    target outside the vocabulary makes its row's loss and gradients NaN."""
    if reduction not in _hip.REDUCTIONS:
        raise RuntimeError(f"reduction must be one of {sorted(_hip.REDUCTIONS)}, got {reduction!r}")
    ops.check_loss(logits, targets)
    if _tracked(logits):
        return _CrossEntropyFn.apply(logits, targets, int(ignore_index), reduction)
    loss, _, _ = ops.loss_forward(*_loss_operands(logits, targets), int(ignore_index), reduction, False)
    return loss.view(targets.shape) if reduction == "none" else loss


def cross_entropy_with_grad(logits: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
                            grad_scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, gradient): the mean cross-entropy and grad_scale times its gradient by logits (shaped and
    typed as they are), from one pass over them. For training loops that start the backward pass at
    the logits: `logits.backward(gradient)`. Arguments as cross_entropy's; not tracked by autograd."""
    ops.check_loss(logits, targets)
    x, t = _loss_operands(logits.detach(), targets)
    loss, grad = ops.loss_with_grad(x, t, int(ignore_index), float(grad_scale))
    return loss, grad.view(logits.shape) if grad.is_contiguous() else grad.reshape(logits.shape)
