"""A transformer block around a physical FFN, on this package's own kernels: pre-norm blocks whose
norms take the residual add along, and attention over a window of tokens and a few first ones,
for training and, with a cache, for generation. The reference's models build these parts of a block
from torch's operators (`nn.LayerNorm`, scaled-dot-product attention).
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn

from isa.kernels.transformer_block import add_layer_norm, layer_norm, window_attention


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over the last dimension (same parameters and state dict) on the HIP kernels."""

    def __init__(self, dim: int, eps: float = 1e-5, bias: bool = True):
        super().__init__(dim, eps=eps, bias=bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)

    def add(self, x: torch.Tensor, residual: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """(norm of x + residual, x + residual)."""
        return add_layer_norm(x, residual, self.weight, self.bias, self.eps)


class WindowCache:
    """The keys and values of a batch's sequences, each of its own length (on the device).

    A caller may set `lengths` (a padded prompt's true ones, or zeros to start anew)."""

    def __init__(self, batch: int, capacity: int, kv_heads: int, head_dim: int, *, dtype=torch.float32, device="cuda"):
        shape = (batch, capacity, kv_heads, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        with torch.inference_mode(False):  # its changes are counted (see longest)
            self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self._rows = torch.arange(batch, device=device)[:, None]
        self._recorded = False  # by a HIP graph, whose replays are not counted
        self._keep(0)

    def _keep(self, longest: int) -> None:
        known = not (self._recorded or self.lengths.is_inference())
        self._longest, self._known = longest, (self.lengths, self.lengths._version if known else None)

    def longest(self) -> Optional[int]:
        """The longest sequence's length; None while a HIP graph is recorded. Kept on the host: the device is
        asked only after a caller set `lengths`, and after a graph recorded an append."""
        if self.lengths.is_cuda and torch.cuda.is_current_stream_capturing():
            self._recorded = True
            return None
        tensor, version = self._known
        if self._recorded or tensor is not self.lengths or version is None or version != self.lengths._version:
            self._keep(int(self.lengths.max()) if self.lengths.numel() else 0)
        return self._longest

    @torch.no_grad()
    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """Adds tokens [batch, n, kv_heads, head_dim] behind each sequence's end, if all fit, without their
        gradients. (Where a HIP graph replays appends, the caller keeps them within the capacity.)"""
        n, used, capacity = k.shape[1], self.longest() or 0, self.k.shape[1]
        if used + n > capacity:
            raise RuntimeError(f"{n} tokens do not fit a cache of {capacity} that holds {used}")
        at = self.lengths.long()[:, None] + torch.arange(n, device=k.device)
        self.k[self._rows, at] = k.to(self.k.dtype)
        self.v[self._rows, at] = v.to(self.v.dtype)
        self.lengths += n
        self._keep(used + n)


class _OverACache(torch.autograd.Function):
    """Attention's output over a cache. A cache holds values alone: a backward pass would leave out what reaches
    a token's key and value through it, so there is none."""

    @staticmethod
    def forward(ctx, out, k, v):
        return out.view_as(out)

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("attention over a WindowCache has no gradients: train without a cache")


class WindowAttention(nn.Module):
    """Causal self-attention over the last `window` tokens and the first `sinks` ones, with a joint
    projection to queries, keys and values (kv_heads of the latter two, shared by the query heads)."""

    def __init__(self, dim: int, heads: int, *, kv_heads: Optional[int] = None, window: Optional[int] = None,
                 sinks: int = 0):
        super().__init__()
        if dim % heads:
            raise ValueError(f"dim ({dim}) must be a multiple of heads ({heads})")
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads or heads, dim // heads
        self.window, self.sinks = window, sinks
        self.qkv = nn.Linear(dim, (heads + 2 * self.kv_heads) * self.head_dim)
        self.proj = nn.Linear(dim, dim)

    def forward(self, x: torch.Tensor, cache: Optional[WindowCache] = None) -> torch.Tensor:
        b, n, _ = x.shape
        joint = self.qkv(x).view(b, n, self.heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = joint.split((self.heads, self.kv_heads, self.kv_heads), dim=2)
        if cache is None:
            a = window_attention(q, k, v, window=self.window, sinks=self.sinks)
        else:
            cache.append(k, v)
            a = window_attention(q.to(cache.k.dtype), cache.k, cache.v, window=self.window, sinks=self.sinks,
                                 key_lengths=cache.lengths)
            if torch.is_grad_enabled():
                a = _OverACache.apply(a, k, v)
        return self.proj(a.reshape(b, n, -1).to(x.dtype))


class Block(nn.Module):
    """Norm, attention, norm, FFN. A branch's output joins the residual stream inside the next norm, so
    a block takes the last one's FFN output and the stream, and returns its own pair."""

    def __init__(self, dim: int, attention: WindowAttention, ffn: nn.Module):
        super().__init__()
        self.ln1, self.attention = LayerNorm(dim), attention
        self.ln2, self.ffn = LayerNorm(dim), ffn

    def forward(self, branch: Optional[torch.Tensor], stream: torch.Tensor, cache: Optional[WindowCache] = None):
        y, stream = (self.ln1(stream), stream) if branch is None else self.ln1.add(branch, stream)
        y, stream = self.ln2.add(self.attention(y, cache), stream)
        return self.ffn(y), stream


class GPT(nn.Module):
    """Token and position embeddings, blocks, a last norm and the tied output projection."""

    def __init__(self, vocab: int, positions: int, dim: int, blocks: nn.ModuleList):
        super().__init__()
        self.tokens = nn.Embedding(vocab, dim)
        self.positions = nn.Embedding(positions, dim)
        self.blocks = blocks
        self.ln_f = LayerNorm(dim)
        for table in (self.tokens, self.positions):  # logits of untrained weights near zero
            nn.init.normal_(table.weight, std=0.02)

    def forward(self, ids: torch.Tensor, caches: Optional[list] = None) -> torch.Tensor:
        """Logits [batch, n, vocab]; with caches (one a block) ids continue their sequences."""
        used, positions = caches[0].longest() or 0 if caches else 0, self.positions.num_embeddings
        if used + ids.shape[1] > positions:
            raise RuntimeError(f"{ids.shape[1]} tokens after {used} do not fit the table of {positions} positions")
        at = torch.arange(ids.shape[1], device=ids.device)
        if caches is not None:
            at = caches[0].lengths.long()[:, None] + at
        branch, stream = None, self.tokens(ids) + self.positions(at)
        for i, block in enumerate(self.blocks):
            branch, stream = block(branch, stream, None if caches is None else caches[i])
        y = self.ln_f(stream) if branch is None else self.ln_f.add(branch, stream)[0]
        return nn.functional.linear(y, self.tokens.weight)

    def caches(self, batch: int, capacity: int, **options) -> list:
        """Empty caches for generation."""
        a = [block.attention for block in self.blocks]
        return [WindowCache(batch, capacity, x.kv_heads, x.head_dim, device=self.tokens.weight.device, **options) for x in a]
