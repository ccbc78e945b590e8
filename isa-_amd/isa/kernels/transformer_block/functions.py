"""The public operators of a transformer block around its FFN and of its training step, with their gradients."""

from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

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


def embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, positions: Optional[torch.Tensor] = None,
              position_weight: Optional[torch.Tensor] = None, padding_index: Optional[int] = None) -> torch.Tensor:
    """scale * weight[ids], and with a second table + position_weight[positions], in one pass: [*ids.shape, dim].

    ids: int64 or int32 of any shape on weight's device; weight: [vocab, dim], position_weight: [places, dim] of its type
    (float32, bfloat16 or float16), at most 2^24 rows and 2^20 columns. positions broadcast to ids; without them the tokens along
    ids' last dimension stand at 0, 1, 2, ... The sum is made in fp32 and rounded once.

    An id or a position outside its table makes its row NaN and takes no part in that table's gradient, nor does
    padding_index in weight's. The gradients (dense, shaped as the tables) are fp32 sums over the tokens sorted by row,
    rounded once, without atomics: the same call gives the same bits."""
    return _binding.embedding(ids, weight, scale, positions, position_weight, padding_index, False)


def unchecked_embedding(ids, weight, *, scale=1.0, positions=None, position_weight=None, padding_index=None) -> torch.Tensor:
    """embedding for a model that calls leaves_can_be_captured in its backward pass: so a forward pass alone can be
    captured whatever graphs of the tables live."""
    return _binding.embedding(ids, weight, scale, positions, position_weight, padding_index, True)


def leaves_can_be_captured(leaves: Sequence[torch.Tensor]) -> None:
    """While a HIP graph is recorded: refuses leaves of which a graph made on the default stream still lives. A backward
    pass that reached one would end the process."""
    _binding.leaves_can_be_captured(list(leaves))


def dropout(x: torch.Tensor, p: float, seed: torch.Tensor, *, site: int = 0) -> torch.Tensor:
    """x with elements dropped (set to 0, whatever they held) with probability p, the others divided by 1 - p.

    No mask is stored: which elements are dropped follows from seed, int64 [2] on x's device (a key and an offset), from
    site, which is added to the offset, and from an element's row and column (x as rows of its last dimension), by
    Philox4x32-10 (Salmon et al. 2011). p is held to a multiple of 2^-16, and the factor follows what it is held to.
    Calls that should differ need another key, offset or site: one training step takes one offset and the next one is
    past its sites. The backward pass reads seed again, so it is not to be changed in place before (autograd says so);
    a HIP graph's replays differ where the graph itself, or its caller, counts the offset up.

    x: float32, bfloat16 or float16, [..., dim]."""
    return _binding.dropout(x, p, seed, site)


def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                           bias: Optional[torch.Tensor] = None, eps: float = 1e-5, *, p: float, seed: torch.Tensor,
                           site: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, h): h = dropout(x) + residual, rounded once to residual's type, and y = layer_norm(h, weight, bias, eps), in
    add_layer_norm's pass. Arguments as add_layer_norm's and dropout's, which drops the same elements."""
    return _binding.dropout_add_layer_norm(x, residual, weight, bias, eps, p, seed, site)


Clip = Union[None, float, Tuple[float, float]]


def _bounds(clip: Clip) -> Tuple[float, float]:
    low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    return 1.0 if low is None else low, float("inf") if high is None else high


def policy_loss(logits: torch.Tensor, actions: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor, *,
                ref_logp: Optional[torch.Tensor] = None, clip: Clip = 0.2, kl: float = 0.0, ignore_index: int = -100,
                reduction: str = "mean") -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, logp): the clipped policy loss of the actions' log-probabilities logp = log softmax(logits)[action],

        -min(r A, clamp(r, 1 - low, 1 + high) A) + kl (exp(ref_logp - logp) - (ref_logp - logp) - 1)

    with r = exp(logp - old_logp) and clip = (low, high), a number for both, or None for no bounds; the second term is
    an estimate of the divergence from a reference model. As float32; logp [...] takes no gradient.

    logits: [..., vocab], float32, bfloat16 or float16; actions: int64 [...]; old_logp, advantages and ref_logp: float32
    [...], held fixed (they must not require a gradient). Rows whose action is ignore_index count nowhere (logp 0);
    reduction is "mean" (over the others), "sum" or "none". Any other action outside the vocabulary makes its row NaN.
    A ratio past a bound on the side that the minimum takes passes no gradient. Rows as cross_entropy's; -cross_entropy
    with reduction "none" gives old_logp and ref_logp."""
    return _binding.policy_loss(logits, actions, old_logp, advantages, ref_logp, *_bounds(clip), kl, ignore_index, reduction)


def policy_loss_with_grad(logits: torch.Tensor, actions: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor, *,
                          ref_logp: Optional[torch.Tensor] = None, clip: Clip = 0.2, kl: float = 0.0,
                          ignore_index: int = -100,
                          grad_scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(loss, gradient, logp): the mean policy loss and grad_scale times its gradient by logits (shaped and typed as they
    are), from one pass over them, for `logits.backward(gradient)`. Arguments as policy_loss's; not tracked by autograd."""
    return _binding.policy_loss_with_grad(logits, actions, old_logp, advantages, ref_logp, *_bounds(clip), kl, ignore_index,
                                          grad_scale)


def preference_loss(logits: torch.Tensor, targets: torch.Tensor, ref_logp: torch.Tensor, *, beta: float = 0.1,
                    ignore_index: int = -100, reduction: str = "mean") -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, logp): the preference loss of pairs of sequences, -log sigmoid(m) with

        m = beta ((logp - ref_logp) of the chosen sequence - (logp - ref_logp) of the rejected one)

    where a sequence's logp is the sum of its targets' log-probabilities (in 64 bits). As float32; logp [2 pairs] takes
    no gradient.

    logits: [2 pairs, tokens, vocab], float32, bfloat16 or float16, the chosen sequences before the rejected ones in the
    same order; targets: int64 [2 pairs, tokens], ignore_index where a token does not count (prompts, padding); ref_logp:
    float32 [2 pairs], the same sums of a reference model, held fixed. reduction is "mean" (over the pairs), "sum" or
    "none" ([pairs]). Any other target outside the vocabulary makes its pair NaN."""
    return _binding.preference_loss(logits, targets, ref_logp, beta, ignore_index, reduction)


def preference_loss_with_grad(logits: torch.Tensor, targets: torch.Tensor, ref_logp: torch.Tensor, *, beta: float = 0.1,
                              ignore_index: int = -100,
                              grad_scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(loss, gradient, logp): the mean preference loss and grad_scale times its gradient by logits (shaped and typed as
    they are), for `logits.backward(gradient)`. Arguments as preference_loss's; not tracked by autograd."""
    return _binding.preference_loss_with_grad(logits, targets, ref_logp, beta, ignore_index, grad_scale)
