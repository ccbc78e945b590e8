"""Dropout and the norm with dropout in its residual add against the generator's definition and the norm's formulas.

Which elements are dropped is exact. A kept one is one fp32 product, rounded: u + v of its size (u of the type,
v = 2^-24), v more for the factor itself, which is rounded to fp32. The norm's tolerances are those of the norm without
dropout: h is exact up to one rounding of either side's sum, y and the gradients u + 64 v in norm.
"""

from __future__ import annotations

import pytest
import torch

from tests.block_helpers import UNIT, close, layer_norm64
from tests.train_helpers import factors

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
V = UNIT[F32]


def seed_on(dev, key=1234567890123, offset=-5):
    return torch.tensor([key, offset], device=dev)


def kept_as(got, x, f, what):
    """got = x f, zeros where f is 0."""
    g, want = got.detach().double().cpu(), x.detach().double().cpu() * f
    assert torch.equal(g[f == 0], torch.zeros_like(g[f == 0])), what
    tiny = 2.0 ** -25 if got.dtype == F16 else 0.0
    assert float(((g - want).abs() - (UNIT[got.dtype] + 3 * V) * want.abs()).max()) <= tiny, what


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (3, 8), (5, 9), (17, 16), (4, 390), (2, 3, 129), (300, 24), (2, 4096)], ids=str)
def test_dropout(cuda_device, shape, dtype):
    from isa.kernels.transformer_block import dropout

    print(f"[case] dropout {shape} {dtype}", flush=True)
    g = torch.Generator(device=cuda_device).manual_seed(sum(shape))
    x, dy = (torch.randn(*shape, generator=g, device=cuda_device).to(dtype) for _ in range(2))
    rows, dim = x.numel() // shape[-1], shape[-1]
    for p, key, offset, site in ((0.1, 7, 0, 0), (0.5, -3, 2 ** 62, 5), (0.999, 2 ** 40 + 9, -1, -7), (0.0, 1, 1, 0), (1.0, 1, 1, 0)):
        f = factors(rows, dim, p, (key, offset), site).view(shape)
        leaf = x.detach().requires_grad_(True)
        y = dropout(leaf, p, seed_on(cuda_device, key, offset), site=site)
        assert y.dtype == dtype and y.shape == x.shape
        kept_as(y, x, f, f"y at {p}")
        (dx,) = torch.autograd.grad(y, leaf, dy)
        kept_as(dx, dy, f, f"dx at {p}")
        with torch.no_grad():
            assert torch.equal(dropout(x, p, seed_on(cuda_device, key, offset), site=site), y)


def test_dropped_elements_are_zero_whatever_they_held(cuda_device):
    from isa.kernels.transformer_block import dropout

    x = torch.full((40, 64), float("nan"), device=cuda_device)
    x[::2] = float("inf")
    y = dropout(x, 0.5, seed_on(cuda_device))
    gone = (factors(40, 64, 0.5, (1234567890123, -5)) == 0).to(cuda_device)
    assert torch.equal(y == 0, gone) and torch.equal(torch.isnan(y), ~gone & torch.isnan(x))


def test_views(cuda_device):
    """What is dropped follows from an element's row and column, not from where it lies."""
    from isa.kernels.transformer_block import dropout

    whole = torch.randn(6, 10, 48, device=cuda_device)
    s = seed_on(cuda_device)
    for name, x in (("columns", whole[:, :, 5:40]), ("rows", whole[:, 2:9]), ("transposed", whole.transpose(0, 1)),
                    ("elements apart", whole[..., ::3]), ("spread", whole[:1, :, :7].expand(6, 10, 7)), ("one row", whole[0, 0])):
        print(f"[case] {name}", flush=True)
        assert torch.equal(dropout(x, 0.3, s), dropout(x.contiguous(), 0.3, s))
        leaf = x.detach().requires_grad_(True)
        up = torch.randn_like(x.contiguous())
        (a,) = torch.autograd.grad(dropout(leaf, 0.3, s), leaf, up)
        assert torch.equal(a, dropout(up, 0.3, s))
        (a,) = torch.autograd.grad(dropout(leaf, 0.3, s).sum(), leaf)
        assert torch.equal(a, dropout(torch.ones_like(up), 0.3, s))
    for shape in ((0, 8), (8, 0), (0,)):
        leaf = torch.zeros(shape, device=cuda_device, requires_grad=True)
        y = dropout(leaf, 0.3, s)
        assert y.shape == shape and torch.autograd.grad(y, leaf, y)[0].shape == shape


def test_changed_seed_is_noticed(cuda_device):
    from isa.kernels.transformer_block import dropout

    leaf, s = torch.randn(4, 8, device=cuda_device, requires_grad=True), seed_on(cuda_device)
    y = dropout(leaf, 0.5, s)
    s += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


# widths of every path: lanes' chunks of 4 and 8, whole waves and blocks, cut vectors
DIMS = [1, 5, 8, 63, 64, 100, 256, 390, 512, 771, 1024, 2048, 2050, 4096, 8192, 9001, 16384]


@pytest.mark.parametrize("types", [(F32, F32, F32), (BF16, F32, F32), (F16, F32, F32), (BF16, BF16, BF16), (F16, F16, F32),
                                   (F16, F16, F16), (BF16, BF16, F32)], ids=str)
def test_norm_with_dropout(cuda_device, types):
    from isa.kernels.transformer_block import add_layer_norm, dropout_add_layer_norm

    xt, st, wt = types
    for dim in DIMS:
        rows = 9 if dim > 1000 else 70
        print(f"[case] dropout norm {rows} x {dim} {types}", flush=True)
        g = torch.Generator(device=cuda_device).manual_seed(dim)
        rnd = lambda *s, to: torch.randn(*s, generator=g, device=cuda_device).to(to)  # noqa: E731
        x, r, dy, dh = rnd(rows, dim, to=xt), rnd(rows, dim, to=st) + 0.5, rnd(rows, dim, to=st), rnd(rows, dim, to=st)
        w, b = 1.0 + 0.2 * rnd(dim, to=wt), rnd(dim, to=wt)
        p, key, offset, site = 0.3, 99 + dim, 2 ** 33, 3
        f = factors(rows, dim, p, (key, offset), site)
        leaves = [t.requires_grad_(True) for t in (x, r, w, b)]
        s = seed_on(cuda_device, key, offset)
        y, h = dropout_add_layer_norm(*leaves, p=p, seed=s, site=site)
        grads = torch.autograd.grad((y, h), leaves, (dy, dh))
        assert y.dtype == h.dtype == st and grads[0].dtype == xt
        # h: the sum in fp32 (two roundings of it), rounded once
        exact = r.detach().double().cpu() + x.detach().double().cpu() * f
        size = r.detach().double().cpu().abs() + (x.detach().double().cpu() * f).abs()
        assert float(((h.detach().double().cpu() - exact).abs() - UNIT[st] * exact.abs() - 3 * V * size).max()) <= 0.0
        want = layer_norm64(h.detach().cpu(), w.detach().cpu(), b.detach().cpu(), 1e-5, dy.cpu(), dh.cpu())
        tol = UNIT[st] + 64 * V
        if dim > 1:  # of one column y is the bias, and its gradients are 0
            close(y, want[0], tol, "y")
            close(grads[1], want[1], tol, "dresidual")
            close(grads[2], want[2], UNIT[wt] + 64 * V + 2e-6, "dweight")
        close(grads[3], want[3], UNIT[wt] + 64 * V, "dbias")
        dx = grads[0].double().cpu()
        assert torch.equal(dx[f == 0], torch.zeros_like(dx[f == 0]))
        close(grads[0], want[1] * f, UNIT[xt] + 64 * V, "dx")
        with torch.no_grad():
            again = dropout_add_layer_norm(x, r, w, b, p=p, seed=s, site=site)
            assert torch.equal(again[0], y) and torch.equal(again[1], h)
            # nothing dropped: the norm without dropout. Its h is the same sum; y's last product and sum may be
            # rounded with the conversion to 16 bits in one kernel and before it in the other
            ours, plain = dropout_add_layer_norm(x, r, w, b, p=0.0, seed=s), add_layer_norm(x, r, w, b)
            assert torch.equal(ours[1], plain[1])
            close(ours[0], plain[0], tol, "y without dropping")


def test_norm_with_dropout_of_views(cuda_device):
    from isa.kernels.transformer_block import dropout, dropout_add_layer_norm

    g = torch.Generator(device=cuda_device).manual_seed(0)
    big = [torch.randn(4, 12, 100, generator=g, device=cuda_device) for _ in range(2)]
    s = seed_on(cuda_device)
    for name, cut in (("columns", lambda t: t[..., 3:67]), ("unaligned", lambda t: t[..., 1:78]), ("rows", lambda t: t[:, ::2]),
                      ("transposed", lambda t: t.transpose(0, 1)), ("elements apart", lambda t: t[..., ::2])):
        print(f"[case] {name}", flush=True)
        x, r = (cut(t) for t in big)
        w = torch.randn(x.shape[-1], generator=g, device=cuda_device)
        a = dropout_add_layer_norm(x, r, w, p=0.25, seed=s)
        b = dropout_add_layer_norm(x.contiguous(), r.contiguous(), w, p=0.25, seed=s)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.equal(a[1], dropout(x, 0.25, s) + r)
    # y's or h's gradient alone, and not every input's
    leaves = [t[0, :, :64].clone().requires_grad_(True) for t in big]
    w = torch.ones(64, device=cuda_device)
    y, h = dropout_add_layer_norm(*leaves, w, p=0.25, seed=s)
    (dx,) = torch.autograd.grad(h.sum(), leaves[0], retain_graph=True)
    assert torch.equal(dx, dropout(torch.ones_like(dx), 0.25, s))
    dx, dr = torch.autograd.grad(y.square().sum(), leaves)
    torch.testing.assert_close(dx, dropout(dr, 0.25, s), rtol=1e-6, atol=1e-7)
    none = dropout_add_layer_norm(*(t[:0] for t in leaves), w, p=0.25, seed=s)
    assert none[0].shape == (0, 64)
