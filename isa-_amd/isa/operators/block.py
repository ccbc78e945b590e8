"""A transformer block around a physical FFN, on this package's own kernels: pre-norm blocks whose
norms take the residual add and its dropout along, attention over a window of tokens and a few first ones,
and embeddings of tokens and positions in one pass, for training and, with a cache, for generation. The reference's models build these parts of a block
from torch's operators (`nn.LayerNorm`, scaled-dot-product attention).
"""

from __future__ import annotations

import inspect
import threading
from numbers import Real
from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch.nn.modules.module import _has_any_global_hook

from isa.kernels.transformer_block import (add_layer_norm, dropout, dropout_add_layer_norm, embedding, layer_norm,
                                           window_attention)
from isa.kernels.transformer_block.functions import leaves_can_be_captured, unchecked_embedding


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over the last dimension (same parameters and state dict) on the HIP kernels."""

    def __init__(self, dim: int, eps: float = 1e-5, bias: bool = True):
        super().__init__(dim, eps=eps, bias=bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)

    def add(self, x: torch.Tensor, residual: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """(norm of x + residual, x + residual)."""
        return add_layer_norm(x, residual, self.weight, self.bias, self.eps)

    def drop_add(self, x: torch.Tensor, residual: torch.Tensor, p: float, seed: torch.Tensor,
                 site: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """The same of dropout(x, p, seed, site=site)."""
        return dropout_add_layer_norm(x, residual, self.weight, self.bias, self.eps, p=p, seed=seed, site=site)


class Embedding(nn.Embedding):
    """nn.Embedding (same parameters and state dict) on the HIP kernels: looked up times `scale`, a padding_idx without
    a gradient. Its other options (max_norm, scale_grad_by_freq, sparse) are refused. An index outside the table makes
    its row NaN."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: Optional[int] = None, *,
                 scale: float = 1.0, **options):
        super().__init__(num_embeddings, embedding_dim, padding_idx, **options)
        if self.max_norm is not None or self.scale_grad_by_freq or self.sparse:
            raise ValueError("max_norm, scale_grad_by_freq and sparse are not supported")
        self.scale = scale

    def forward(self, ids: torch.Tensor, positions: Optional[torch.Tensor] = None,
                position_weight: Optional[torch.Tensor] = None, *, operator=None) -> torch.Tensor:
        """With a table of positions (a place of its own for each token of a sequence unless `positions` are given)
        the sum of both. operator: `embedding` unless given."""
        return (operator or embedding)(ids, self.weight, scale=self.scale, positions=positions,
                                       position_weight=position_weight, padding_index=self.padding_idx)


def _is_ours(table: nn.Module) -> bool:
    return type(table) is Embedding and "forward" not in vars(table)


def _operator_alone(table: nn.Module) -> bool:
    """Whether a call of this table is `embedding` of its weight and nothing else: no hooks, no forward of a caller's."""
    return (_is_ours(table) and not _has_any_global_hook() and not (
        table._forward_hooks or table._forward_pre_hooks or table._backward_hooks or table._backward_pre_hooks))


_ONE_STEP = threading.Lock()  # (of all seeds: one of its own could not be copied or pickled with a model)


class DropoutSeed:
    """The key and offset of a model's dropout, an int64 tensor [2] that moves to the device of the steps.

    A forward pass takes `step`: a copy for its calls, whose sites are 0 .. sites - 1, while the offset moves past them,
    on the device, so that a HIP graph that recorded a step draws anew in each replay; the first step on a device, which
    moves the state there, comes before any that is captured. Steps of several threads or streams come one after the
    other; a graph's replays are ordered by who replays it.

    key: drawn from torch's generator unless given; ranks of one job take a key each. (Not a buffer of the model: those
    are made alike on all ranks, so no state dict has it. A run that is to go on where it stopped keeps `state` with its
    checkpoint and copies it back; one that starts again under the same torch.manual_seed repeats its first masks.)"""

    _stream = _done = None  # of the last eager step on a GPU, and its end

    def __init__(self, key: Optional[int] = None):
        with torch.inference_mode(False):  # it changes in place, in any mode
            self.state = torch.tensor([int(torch.randint(2 ** 62, ())) if key is None else key, 0])

    def __getstate__(self) -> dict:
        return {k: v for k, v in vars(self).items() if k not in ("_stream", "_done")}

    def _wait(self) -> None:
        if self._done is not None and self.state.is_cuda:
            stream = torch.cuda.current_stream(self.state.device)
            if stream != self._stream:
                stream.wait_event(self._done)

    @torch.no_grad()
    def step(self, sites: int, device: torch.device) -> torch.Tensor:
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        recorded = device.type == "cuda" and torch.cuda.is_current_stream_capturing()
        with _ONE_STEP, torch.inference_mode(False):
            if not recorded:
                self._wait()
            if self.state.device != device:
                # a recorded copy would read memory that is free by then, and set the offset back, in each replay
                if recorded:
                    raise RuntimeError(f"a dropout seed on {self.state.device} cannot move to {device} in a capture: take "
                                       "a step there before one is captured")
                self.state = self.state.to(device)
            seed = self.state.clone()
            self.state[1:].add_(sites)
            if device.type == "cuda" and not recorded:
                stream = torch.cuda.current_stream(device)
                if self._done is None or self._stream.device != stream.device:
                    self._done = torch.cuda.Event()
                self._done.record(stream)
                self._stream = stream
        return seed


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


def _join(norm: LayerNorm, branch: torch.Tensor, stream: torch.Tensor, p: float, seed: Optional[torch.Tensor], site: int):
    if seed is None or p == 0.0:
        return norm.add(branch, stream)
    return norm.drop_add(branch, stream, p, seed, site)


class Block(nn.Module):
    """Norm, attention, norm, FFN. A branch's output joins the residual stream inside the next norm, so
    a block takes the last one's FFN output and the stream, and returns its own pair.

    With `dropout` and a seed (`DropoutSeed.step`; none: no dropout) a block that trains (its own flag says so) drops the
    branches' outputs as they join: the last block's under `site`, the own attention's under site + 1."""

    def __init__(self, dim: int, attention: WindowAttention, ffn: nn.Module, dropout: float = 0.0):
        super().__init__()
        self.ln1, self.attention = LayerNorm(dim), attention
        self.ln2, self.ffn = LayerNorm(dim), ffn
        self.dropout = dropout

    def forward(self, branch: Optional[torch.Tensor], stream: torch.Tensor, cache: Optional[WindowCache] = None,
                seed: Optional[torch.Tensor] = None, site: int = 0):
        if not self.training:
            seed = None
        y, stream = (self.ln1(stream), stream) if branch is None else _join(self.ln1, branch, stream, self.dropout, seed, site)
        y, stream = _join(self.ln2, self.attention(y, cache), stream, self.dropout, seed, site + 1)
        return self.ffn(y), stream


def _drops(part: nn.Module) -> bool:
    p = getattr(part, "dropout", 0.0)  # of a caller's block: perhaps a module
    return part.training and isinstance(p, Real) and p != 0.0


def _takes_seed(block: nn.Module) -> bool:
    if type(block) is Block:
        return True
    parameters = inspect.signature(block.forward).parameters.values()
    return any(p.name == "seed" or p.kind is p.VAR_KEYWORD for p in parameters)


class GPT(nn.Module):
    """Token and position embeddings, blocks, a last norm and the tied output projection. `dropout` is that of the
    embeddings and of the last block's output (the blocks have their own), while the model trains (its own flag, and the
    blocks' for theirs); its numbers follow from `seed`, a DropoutSeed that the model makes when it first drops unless the
    caller sets one. Blocks of a caller's own whose forward has no `seed` get none."""

    def __init__(self, vocab: int, positions: int, dim: int, blocks: nn.ModuleList, dropout: float = 0.0):
        super().__init__()
        self.tokens = Embedding(vocab, dim)
        self.positions = Embedding(positions, dim)
        self.blocks = blocks
        self.ln_f = LayerNorm(dim)
        self.dropout = dropout
        self.seed = None
        for table in (self.tokens, self.positions):  # logits of untrained weights near zero
            nn.init.normal_(table.weight, std=0.02)

    def _step(self, device: torch.device) -> Optional[torch.Tensor]:
        """This pass's seed, if any part drops. Sites: the embeddings', two a block, the last block's output."""
        if not (_drops(self) or any(_drops(block) and _takes_seed(block) for block in self.blocks)):
            return None
        if self.seed is None:
            self.seed = DropoutSeed()
        return self.seed.step(2 + 2 * len(self.blocks), device)

    def _embed(self, ids: torch.Tensor, at: Optional[torch.Tensor], captured: bool = False) -> torch.Tensor:
        tokens, positions = self.tokens, self.positions
        how = [{"operator": unchecked_embedding} if captured and _is_ours(table) else {} for table in (tokens, positions)]
        if (_operator_alone(tokens) and _operator_alone(positions) and positions.scale == 1.0
                and positions.padding_idx is None and tokens.weight.dtype == positions.weight.dtype):
            return tokens(ids, at, positions.weight, **how[0])
        if at is None:  # a caller's own modules, or tables that do more than one call of the operator does
            at = torch.arange(ids.shape[1], device=ids.device)
        return tokens(ids, **how[0]) + positions(at, **how[1])

    def forward(self, ids: torch.Tensor, caches: Optional[list] = None) -> torch.Tensor:
        """Logits [batch, n, vocab]; with caches (one a block) ids continue their sequences."""
        used, positions = caches[0].longest() or 0 if caches else 0, self.positions.num_embeddings
        if used + ids.shape[1] > positions:
            raise RuntimeError(f"{ids.shape[1]} tokens after {used} do not fit the table of {positions} positions")
        at = None
        if caches is not None:
            at = caches[0].lengths.long()[:, None] + torch.arange(ids.shape[1], device=ids.device)
        seed = self._step(ids.device)
        captured = ids.is_cuda and torch.is_grad_enabled() and torch.cuda.is_current_stream_capturing()
        branch, stream = None, self._embed(ids, at, captured)
        p = self.dropout if self.training else 0.0
        if seed is not None and p:
            stream = dropout(stream, p, seed)
        for i, block in enumerate(self.blocks):
            rest = {"seed": seed, "site": 1 + 2 * i} if seed is not None and _takes_seed(block) else {}
            branch, stream = block(branch, stream, None if caches is None else caches[i], **rest)
        if branch is None:
            y = self.ln_f(stream)
        else:
            y = _join(self.ln_f, branch, stream, p, seed, 1 + 2 * len(self.blocks))[0]
        logits = nn.functional.linear(y, self.tokens.weight)
        if captured and logits.requires_grad:  # a forward pass may be captured beside any graph; a backward may not
            logits.register_hook(lambda _: leaves_can_be_captured(self.parameters()))
        return logits

    def caches(self, batch: int, capacity: int, **options) -> list:
        """Empty caches for generation."""
        a = [block.attention for block in self.blocks]
        return [WindowCache(batch, capacity, x.kv_heads, x.head_dim, device=self.tokens.weight.device, **options) for x in a]
