"""Operators of a transformer block around its FFN and of its training step (HIP, gfx950): layer norm with the residual
add, attention with a sliding window and sinks, embeddings, dropout, and the cross-entropy, policy and preference
losses, with their gradients. The reference runs these on torch's own operators."""

from isa.kernels.transformer_block.functions import (
    add_layer_norm,
    cross_entropy,
    cross_entropy_with_grad,
    dropout,
    dropout_add_layer_norm,
    embedding,
    layer_norm,
    policy_loss,
    policy_loss_with_grad,
    preference_loss,
    preference_loss_with_grad,
    window_attention,
)

__all__ = ["add_layer_norm", "cross_entropy", "cross_entropy_with_grad", "dropout", "dropout_add_layer_norm", "embedding",
           "layer_norm", "policy_loss", "policy_loss_with_grad", "preference_loss", "preference_loss_with_grad",
           "window_attention"]
