"""The block's modules against the same block of torch's operators, and the example that trains a
small GPT with them and generates from it."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from tests.block_helpers import close, visible
from tests.helpers import flash_cfg

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "isa-_amd" / "examples"))


def plain_block(block, x):
    """Block.forward of torch's operators; returns the stream after the block."""
    a = block.attention
    b, n, d = x.shape
    y = F.layer_norm(x, (d,), block.ln1.weight, block.ln1.bias, block.ln1.eps)
    joint = F.linear(y, a.qkv.weight, a.qkv.bias).view(b, n, -1, a.head_dim)
    q, k, v = joint.split((a.heads, a.kv_heads, a.kv_heads), dim=2)
    k, v = (t.repeat_interleave(a.heads // a.kv_heads, 2).transpose(1, 2).contiguous() for t in (k, v))
    s = torch.matmul(q.transpose(1, 2), k.transpose(2, 3).contiguous()) / a.head_dim ** 0.5
    hidden = ~visible(1, n, n, a.window, a.sinks, None).to(x.device)
    o = torch.matmul(torch.softmax(s.masked_fill(hidden, float("-inf")), -1), v).transpose(1, 2).reshape(b, n, d)
    x = x + F.linear(o, a.proj.weight, a.proj.bias)
    return x + block.ffn(F.layer_norm(x, (d,), block.ln2.weight, block.ln2.bias, block.ln2.eps))


def make_block(dev, ffn, dim=96, heads=6, kv_heads=2, window=20, sinks=3):
    from isa.operators.block import Block, WindowAttention

    torch.manual_seed(0)
    return Block(dim, WindowAttention(dim, heads, kv_heads=kv_heads, window=window, sinks=sinks), ffn).to(dev)


def test_block_matches_torch(cuda_device):
    """fp32 in two orders of summation through a norm, an attention and an FFN: some 100 roundings of 2^-24."""
    from isa.operators.cim import PhysicalFFN

    ffn = PhysicalFFN(96, 192, flash_cfg(4096))
    ffn.fc1.set_r_tia(1e6)
    block = make_block(cuda_device, ffn)
    x = torch.randn(3, 70, 96, device=cuda_device)
    g = torch.randn_like(x)

    def run(f):
        block.zero_grad(set_to_none=True)
        leaf = x.clone().requires_grad_(True)
        out = f(leaf)
        out.backward(g)
        return [out.detach(), leaf.grad] + [p.grad.clone() for p in block.attention.parameters()] + [
            block.ln1.weight.grad.clone(), block.ln2.bias.grad.clone()]

    def ours(leaf):
        branch, stream = block(None, leaf)
        return branch + stream

    for i, (a, b) in enumerate(zip(run(ours), run(lambda leaf: plain_block(block, leaf)))):
        close(a, b, 2e-5, f"output {i}")


def test_state_dict_is_torchs(cuda_device):
    from isa.operators.block import LayerNorm

    a, b = LayerNorm(64).to(cuda_device), nn.LayerNorm(64).to(cuda_device)
    with torch.no_grad():
        b.weight.normal_()
        b.bias.normal_()
    a.load_state_dict(b.state_dict())
    x = torch.randn(5, 64, device=cuda_device)
    close(a(x), b(x), 1e-6, "layer norm")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_block_under_autocast(cuda_device, dtype):
    """Projections and attention in 16 bits, the stream and its norms in fp32: within a few roundings of the
    16-bit type (u) of the fp32 block's branch outputs, which are a fraction of the stream."""
    from tests.block_helpers import UNIT

    block = make_block(cuda_device, nn.Identity())
    x = torch.randn(2, 50, 96, device=cuda_device)
    _, plain = block(None, x)
    with torch.autocast("cuda", dtype=dtype):
        leaf = x.clone().requires_grad_(True)
        branch, stream = block(None, leaf)
    assert stream.dtype == torch.float32 and branch.dtype == torch.float32
    close(stream, plain, 8 * UNIT[dtype], "stream")
    (branch + stream).sum().backward()
    assert torch.isfinite(leaf.grad).all() and all(torch.isfinite(p.grad).all() for p in block.parameters())


def test_example_trains_and_generates(cuda_device):
    import window_gpt

    torch.manual_seed(0)
    generator = torch.Generator(device="cuda").manual_seed(0)
    model = window_gpt.make_model()
    losses = window_gpt.train(model, 150, generator)
    print(f"losses: {losses[0]:.3f} ... {losses[-1]:.3f}", flush=True)
    assert losses[-1] < 0.5 * losses[0]
    # what single tokens over the cache give is what the whole sequence gives
    prompt = window_gpt.batch(3, 40, generator)
    ids, logits = window_gpt.generate(model, prompt, 30)
    with torch.no_grad():
        whole = model(ids[:, :-1])[:, prompt.shape[1] - 1:]
    close(logits, whole, 1e-4, "logits over the cache")
    with pytest.raises(RuntimeError, match="do not fit"):
        model.caches(1, 8)[0].append(torch.zeros(1, 9, 2, 32, device=cuda_device), torch.zeros(1, 9, 2, 32, device=cuda_device))
