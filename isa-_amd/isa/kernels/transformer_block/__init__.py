"""Operators of a transformer block around its FFN (HIP, gfx950): layer norm with the residual
add, attention with a sliding window and sinks, and the cross-entropy, with their gradients.
The reference runs these on torch's own operators."""

from isa.kernels.transformer_block.functions import (
    add_layer_norm,
    cross_entropy,
    cross_entropy_with_grad,
    layer_norm,
    window_attention,
)

__all__ = ["add_layer_norm", "cross_entropy", "cross_entropy_with_grad", "layer_norm", "window_attention"]
