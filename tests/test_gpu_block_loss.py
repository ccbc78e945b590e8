"""The cross-entropy and its gradient against their formulas in 64 bits.

Tolerances (u of the result's type, v = 2^-24): a row's loss is a difference of numbers up to some
20 around it, 64 v of the largest; its gradient an exponential of a difference of up to some 20,
relative error 20 v and some, and one rounding: u + 64 v.
"""

from __future__ import annotations

import math

import pytest
import torch

from tests.block_helpers import UNIT, close, cross_entropy64

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
V = UNIT[F32]


def make(dev, rows, vocab, dtype, seed=0, ignore=-100):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g, device=dev) * 3.0).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device=dev)
    if rows > 2:
        t[1::3] = ignore
    return x, t


# 16-byte chunks of 1 to 16 a thread and more, rows that start at any address
SIZES = [(1, 1), (3, 2), (5, 100), (7, 1023), (4, 4096), (9, 5003), (6, 8192), (5, 16384), (4, 20001), (3, 28672),
         (5, 33333), (3, 50304), (2, 50305), (2, 65536), (3, 70001), (2, 131072), (2, 150001), (300, 257)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_matches_formulas(cuda_device, size, dtype):
    from isa.kernels.transformer_block import cross_entropy, cross_entropy_with_grad

    print(f"[case] loss {size} {dtype}", flush=True)
    x, t = make(cuda_device, *size, dtype, seed=sum(size))
    row, grad = cross_entropy64(x, t, -100)
    count = int((t != -100).sum())
    scale = max(1.0, float(row.abs().max()), float(x.abs().max()))
    # a 16-bit gradient also loses what is below its type's smallest number
    tiny = 2.0 ** -25 if dtype == F16 else 0.0
    tol = UNIT[dtype] + 64 * V

    def grads_close(got, want, what):
        floor = tiny * math.sqrt(want.numel()) / max(float(want.norm()), 1e-30)
        close(got, want, tol + floor, what)

    for reduction, factor, want in (("mean", 1.0 / count, row.sum() / count), ("sum", 1.0, row.sum()), ("none", 1.0, row)):
        leaf = x.detach().requires_grad_(True)
        loss = cross_entropy(leaf, t, reduction=reduction)
        assert loss.dtype == F32
        many = size[0] if reduction == "sum" else 1
        assert float((loss.double().cpu() - want).abs().max()) <= 64 * V * scale * many, reduction
        up = torch.full_like(loss, 0.5)
        (dx,) = torch.autograd.grad(loss, leaf, up)
        assert dx.dtype == dtype
        if float(grad.abs().max()) > 0:
            grads_close(dx, grad * 0.5 * factor, reduction)
        with torch.no_grad():
            assert torch.equal(cross_entropy(x, t, reduction=reduction), loss)
    loss, dx = cross_entropy_with_grad(x, t, grad_scale=8.0)
    assert abs(float(loss) - float(row.sum() / count)) <= 64 * V * scale
    if float(grad.abs().max()) > 0:
        grads_close(dx, grad * (8.0 / count), "one pass")
    assert torch.count_nonzero(dx[t == -100]) == 0


def test_rows_apart_and_shapes(cuda_device):
    """A padded vocabulary's head, elements apart, rows at odd addresses, more dimensions."""
    from isa.kernels.transformer_block import cross_entropy, cross_entropy_with_grad

    for dtype in (F32, BF16):
        whole, t = make(cuda_device, 24, 1031, dtype, seed=3)
        t = t % 500
        for k, x in enumerate((whole[:, :1000], whole[:, 1:1002], whole[:, ::2], whole[::2, 5:505], whole.view(4, 6, 1031))):
            print(f"[case] view {k} {dtype}", flush=True)
            y = t[::2] if k == 3 else t.view(4, 6) if k == 4 else t
            copy = x.contiguous().clone()
            la, da = cross_entropy_with_grad(x, y)
            lb, db = cross_entropy_with_grad(copy, y)
            assert da.shape == x.shape
            close(da, db, 2 * UNIT[dtype] + 64 * V, "gradient")
            assert abs(float(la) - float(lb)) <= 128 * V * float(lb)
            leaf = x.detach().requires_grad_(True)
            (dc,) = torch.autograd.grad(cross_entropy(leaf, y), leaf)
            close(dc, db, 2 * UNIT[dtype] + 128 * V, "autograd")
        # the second half of a padded row is not written
        pad = torch.full((3, 1056), 7.0, dtype=dtype, device=cuda_device)
        before = pad.clone()
        cross_entropy_with_grad(pad[:, :1000], torch.tensor([1, 2, 3], device=cuda_device))
        assert torch.equal(pad, before)


def test_masked_and_infinite_logits(cuda_device):
    from isa.kernels.transformer_block import cross_entropy_with_grad

    for dtype in (F32, BF16, F16):
        print(f"[case] masked logits {dtype}", flush=True)
        x, t = make(cuda_device, 6, 3001, dtype, seed=5, ignore=-100)
        t = t.clamp(0, 99)
        x[:, 100:2000] = -math.inf
        x[:, 2000:] = torch.finfo(dtype).min
        loss, dx = cross_entropy_with_grad(x, t)
        row, grad = cross_entropy64(x[:, :100], t, -100)
        assert abs(float(loss) - float(row.mean())) <= 256 * V * 20
        close(dx[:, :100], grad / 6, UNIT[dtype] + 64 * V + (2.0 ** -20 if dtype == F16 else 0), "gradient")
        assert torch.count_nonzero(dx[:, 100:]) == 0
        # a masked target: its loss is infinite, its gradient is not
        t[0] = 500
        loss, dx = cross_entropy_with_grad(x, t)
        assert float(loss) == math.inf and torch.isfinite(dx).all()


def test_targets_out_of_range_and_all_ignored(cuda_device):
    from isa.kernels.transformer_block import cross_entropy, cross_entropy_with_grad

    x, t = make(cuda_device, 5, 77, F32)
    t = t.clamp(min=0)
    for bad in (77, -1, 2 ** 40, -2 ** 40):
        t[2] = bad
        print(f"[case] target {bad}", flush=True)
        rows = cross_entropy(x, t, reduction="none")
        assert math.isnan(float(rows[2])) and torch.isfinite(rows[[0, 1, 3, 4]]).all()
        loss, dx = cross_entropy_with_grad(x, t)
        assert math.isnan(float(loss)) and torch.isnan(dx[2]).all() and torch.isfinite(dx[[0, 1, 3, 4]]).all()
    t[:] = 9
    loss, dx = cross_entropy_with_grad(x, t, ignore_index=9)
    assert math.isnan(float(loss)) and torch.count_nonzero(dx) == 0
    assert float(cross_entropy(x, t, ignore_index=9, reduction="sum")) == 0.0
    x[1] = math.nan  # an ignored row may hold anything
    assert float(cross_entropy(x, t, ignore_index=9, reduction="sum")) == 0.0
    empty = cross_entropy(x[:0], t[:0], reduction="none")
    assert empty.shape == (0,)
    assert float(cross_entropy(x[:0], t[:0], reduction="sum")) == 0.0


def test_gradient_against_differences(cuda_device):
    """Central differences along a random direction in fp32: steps of 1e-2, some 1e-4 of its size."""
    from isa.kernels.transformer_block import cross_entropy, cross_entropy_with_grad

    x, t = make(cuda_device, 40, 300, F32, seed=6)
    _, dx = cross_entropy_with_grad(x, t)
    step = torch.randn(x.shape, generator=torch.Generator(device=cuda_device).manual_seed(7), device=cuda_device)
    rows = [cross_entropy(x + s * 1e-2 * step, t, reduction="none").double().sum() for s in (1.0, -1.0)]
    difference = float(rows[0] - rows[1]) / 2e-2 / int((t != -100).sum())
    gradient = float((dx.double() * step.double()).sum())
    assert abs(difference - gradient) <= 2e-3 * max(abs(gradient), float(dx.double().norm()))


def test_offsets_past_32_bits(cuda_device):
    from isa.kernels.transformer_block import cross_entropy_with_grad

    rows, vocab = 43_000, 50304
    assert rows * vocab > 2 ** 31
    print("[case] offsets past 2^31", flush=True)
    x = torch.zeros(rows, vocab, dtype=BF16, device=cuda_device)
    t = torch.full((rows,), -100, device=cuda_device)
    last, tt = make(cuda_device, 2, vocab, BF16)
    x[-2:], t[-2:] = last, tt
    loss, dx = cross_entropy_with_grad(x, t)
    row, grad = cross_entropy64(last, tt, -100)
    assert abs(float(loss) - float(row.mean())) <= 64 * V * 20
    close(dx[-2:], grad / 2, UNIT[BF16] + 64 * V, "last rows")
    assert torch.count_nonzero(dx[:-2]) == 0


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_bits_repeat_on_any_stream(cuda_device, dtype):
    from isa.kernels.transformer_block import cross_entropy_with_grad

    x, t = make(cuda_device, 500, 5003, dtype)
    first = cross_entropy_with_grad(x, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = cross_entropy_with_grad(x, t)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_graph_replays(cuda_device):
    from isa.kernels.transformer_block import cross_entropy_with_grad

    x, t = make(cuda_device, 64, 5000, BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cross_entropy_with_grad(x, t)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, dx = cross_entropy_with_grad(x, t)
    for i in range(4):
        print(f"[case] replay {i}", flush=True)
        x.copy_(torch.randn_like(x) * (i + 1))
        t.copy_(torch.randint(0, 5000, t.shape, device=cuda_device))
        graph.replay()
        torch.cuda.synchronize()
        want = cross_entropy_with_grad(x, t)
        assert torch.equal(loss, want[0]) and torch.equal(dx, want[1])


def test_refusals(cuda_device):
    from isa.kernels.transformer_block import cross_entropy, cross_entropy_with_grad

    x, t = make(cuda_device, 4, 10, F32)

    def refused(match, f, *args, **more):
        with pytest.raises(RuntimeError, match=match):
            f(*args, **more)

    for f in (cross_entropy, cross_entropy_with_grad):
        refused("CUDA", f, x.cpu(), t)
        refused("must be float32", f, x.double(), t)
        refused("targets must be int64", f, x, t.int())
        refused("targets must be int64", f, x, t[:3])
        refused("targets must be on", f, x, t.cpu())
    refused("reduction", cross_entropy, x, t, reduction="max")
