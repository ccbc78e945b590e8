"""The public operators of a transformer block around its FFN, with their gradients."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from isa.kernels.transformer_block import _hip

_binding = _hip.load()


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension (at most 16384
    elements), in x's type, with statistics in fp32.

    x: float32, bfloat16 or float16; weight and bias: x's type or float32. First derivatives only, and
    by reverse mode: an input with a forward-mode tangent is refused, and so are traces (torch.jit.trace, make_fx).
    So it is with all operators here."""
    return _binding.layer_norm(x, weight, bias, eps)


def add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                   bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, h): h = x + residual, rounded to residual's type, and y = layer_norm(h, weight, bias, eps).

    x is a branch's output, residual the stream it joins: of one type, or a 16-bit x beside a
    float32 residual (autocast). One pass forward and one backward, which takes the gradient
    that reaches h past the norm along."""
    return _binding.add_layer_norm(x, residual, weight, bias, eps)


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

    Softmax and sums are fp32; scale is 1 / sqrt(head_dim) unless given. Scores may have any finite size;
    but where a row's highest one times scale passes 2^23, its gradients are made of that score's rounding
    and may be infinite or NaN. In 16-bit types the weights
    p, and in the backward p and ds, are rounded to that type for the matrix cores. Of a key that some
    but not all queries of a tile see, an infinity or NaN in v reaches the others too."""
    return _binding.window_attention(q, k, v, window, sinks, scale, key_lengths)


def cross_entropy(logits: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
                  reduction: str = "mean") -> torch.Tensor:
    """-log softmax(logits)[target] over the last dimension, as float32.

    logits: [..., vocab], float32, bfloat16 or float16; targets: int64 [...]. Rows whose target is
    ignore_index count nowhere; reduction is "mean" (over the others), "sum" or "none". Any other
    target outside the vocabulary makes its row's loss and gradients NaN.

    Rows may lie apart (a padded vocabulary, a sequence's last tokens). Leading dimensions that no single
    stride spans are copied first: instead of logits[:, :-1] of several sequences, take all of the logits and
    targets whose last column is ignore_index."""
    return _binding.cross_entropy(logits, targets, ignore_index, reduction)


def cross_entropy_with_grad(logits: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
                            grad_scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, gradient): the mean cross-entropy and grad_scale times its gradient by logits (shaped and
    typed as they are), from one pass over them. For training loops that start the backward pass at
    the logits: `logits.backward(gradient)`. Arguments as cross_entropy's; not tracked by autograd."""
    return _binding.cross_entropy_with_grad(logits, targets, ignore_index, grad_scale)
