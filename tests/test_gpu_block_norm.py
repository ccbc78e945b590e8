"""layer_norm and add_layer_norm against their formulas in 64 bits.

Tolerances (2-norm of the error over the result's, u of the result's type, v = 2^-24): y and dh are
a few fp32 operations and one rounding, u + 16 v; the gradients of weight and bias sum over the rows
in fp32 in a few hundred partial sums, u + 64 v.
"""

from __future__ import annotations

import pytest
import torch

from tests.block_helpers import UNIT, close, layer_norm64

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
V = UNIT[F32]


def make(dev, shape, x_dtype, dtype, w_dtype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    n = shape[-1]
    return {"x": (rnd(*shape) * 0.5).to(x_dtype), "r": (rnd(*shape) + 0.5 * rnd(n)).to(dtype),
            "w": (1.0 + 0.2 * rnd(n)).to(w_dtype), "b": (0.1 * rnd(n)).to(w_dtype), "dy": rnd(*shape).to(dtype),
            "dh": rnd(*shape).to(dtype)}


TYPES = [(F32, F32, F32), (BF16, F32, F32), (F16, F32, F32), (BF16, BF16, BF16), (BF16, BF16, F32), (F16, F16, F16),
         (F16, F16, F32)]
SHAPES = [(1, 1), (3, 7), (1, 768), (5, 64), (130, 192), (65, 256), (33, 390), (2, 9, 768), (1000, 384), (17, 1000),
          (9, 1024), (11, 1537), (10, 2048), (7, 2056), (5, 4096), (4, 4100), (3, 8192), (3, 8200), (2, 16384),
          (2, 16383), (0, 64), (2049, 48)]


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_add_layer_norm(cuda_device, shape, types):
    from isa.kernels.transformer_block import add_layer_norm

    print(f"[case] add_layer_norm {shape} {types}", flush=True)
    i = make(cuda_device, shape, *types, seed=sum(shape))
    leaves = [i[k].requires_grad_(True) for k in ("x", "r", "w", "b")]
    y, h = add_layer_norm(*leaves, 1e-5)
    dx, dr, dw, db = torch.autograd.grad((y, h), leaves, (i["dy"], i["dh"]))
    with torch.no_grad():
        y0, h0 = add_layer_norm(*leaves, 1e-5)
    assert torch.equal(y0, y) and torch.equal(h0, h)
    stored = (i["x"].detach().float() + i["r"].detach().float()).to(types[1])
    assert torch.equal(h.detach(), stored) and h.dtype == y.dtype == types[1]
    if not y.numel():
        assert torch.count_nonzero(dw) == 0 and torch.count_nonzero(db) == 0
        return
    wy, wdh, wdw, wdb = layer_norm64(stored, leaves[2].detach(), leaves[3].detach(), 1e-5, i["dy"], i["dh"])
    u, ux, uw = UNIT[types[1]], UNIT[types[0]], UNIT[types[2]]
    close(y, wy, u + 16 * V, "y")
    close(dr, wdh, u + 16 * V, "dresidual")
    close(dx, wdh, ux + 16 * V, "dx")
    if shape[-1] == 1:  # n is 0
        assert torch.count_nonzero(dw) == 0
    else:
        close(dw, wdw, uw + 64 * V, "dweight")
    close(db, wdb, uw + 64 * V, "dbias")
    assert dx.dtype == types[0] and dr.dtype == types[1] and dw.dtype == db.dtype == types[2]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("shape", [(1, 768), (77, 130), (3, 5, 2050)], ids=str)
def test_layer_norm(cuda_device, shape, dtype):
    from isa.kernels.transformer_block import layer_norm

    print(f"[case] layer_norm {shape} {dtype}", flush=True)
    i = make(cuda_device, shape, dtype, dtype, dtype, seed=1)
    for bias in (None, i["b"]):
        leaves = [t.detach().requires_grad_(True) for t in (i["r"], i["w"], bias) if t is not None]
        y = layer_norm(*leaves, eps=1e-3)
        grads = torch.autograd.grad(y, leaves, i["dy"])
        want = layer_norm64(i["r"], i["w"], bias, 1e-3, i["dy"])
        u = UNIT[dtype]
        close(y, want[0], u + 16 * V, "y")
        for got, w, tol in zip(grads, want[1:], (u + 16 * V, u + 64 * V, u + 64 * V)):
            close(got, w, tol, "gradient")


def test_strides_and_alignment(cuda_device):
    """Rows apart, elements apart, rows at odd addresses, rows repeated: all as their copies."""
    from isa.kernels.transformer_block import add_layer_norm, layer_norm

    g = torch.Generator(device=cuda_device).manual_seed(4)
    for dtype in (F32, BF16):
        wide = torch.randn(40, 800, generator=g, device=cuda_device).to(dtype)
        w = torch.randn(385, generator=g, device=cuda_device).to(dtype)
        views = [wide[:, :384], wide[:, 3:387], wide[:, 0:768:2], wide[::3, 8:392], wide[:1, :384].expand(40, 384),
                 wide[:, :384].t().contiguous().t(), wide.view(5, 8, 800)[:, :, 16:400]]
        for k, v in enumerate(views):
            for weight in (w[:384], w[1:]):
                print(f"[case] view {k} {dtype}", flush=True)
                copy = v.contiguous().clone()
                leaf, leaf_copy = v.detach().requires_grad_(True), copy.requires_grad_(True)
                a, b = layer_norm(leaf, weight), layer_norm(leaf_copy, weight.clone())
                close(a, b, 2 * UNIT[dtype] + 32 * V, "y")
                dy = torch.randn(v.shape, generator=g, device=cuda_device).to(dtype)
                (da,), (dc,) = torch.autograd.grad(a, leaf, dy), torch.autograd.grad(b, leaf_copy, dy)
                close(da, dc, 2 * UNIT[dtype] + 32 * V, "gradient")
                y1, h1 = add_layer_norm(v, copy.detach(), weight)
                y2, h2 = add_layer_norm(copy.detach(), copy.detach(), weight.clone())
                assert torch.equal(h1, h2)
                close(y1, y2, 2 * UNIT[dtype] + 32 * V, "y of the sum")


def test_gradients_that_are_not_asked_for(cuda_device):
    from isa.kernels.transformer_block import add_layer_norm

    i = make(cuda_device, (30, 100), F32, F32, F32)
    want = layer_norm64(i["x"] + i["r"], i["w"], i["b"], 1e-5, i["dy"])
    through = layer_norm64(i["x"] + i["r"], i["w"], i["b"], 1e-5, torch.zeros_like(i["dy"]), i["dh"])
    for asked in ("x", "r", "w", "b", "xw"):
        print(f"[case] gradients {asked}", flush=True)
        t = {k: i[k].detach().clone().requires_grad_(k in asked) for k in ("x", "r", "w", "b")}
        y, _ = add_layer_norm(t["x"], t["r"], t["w"], t["b"])
        y.backward(i["dy"])
        for k, w in zip("xrwb", (want[1], want[1], want[2], want[3])):
            assert (t[k].grad is not None) == (k in asked)
            if k in asked:
                close(t[k].grad, w, 128 * V, k)
    x = i["x"].detach().clone().requires_grad_(True)  # only the stream is used
    _, h = add_layer_norm(x, i["r"], i["w"], i["b"])
    h.backward(i["dh"])
    close(x.grad, through[1], 32 * V, "the stream alone")


def test_gradient_against_differences(cuda_device):
    """Central differences along random directions in fp32: steps of 1e-2 leave some 1e-4 of the
    derivative's size in truncation and rounding."""
    from isa.kernels.transformer_block import add_layer_norm

    i = make(cuda_device, (20, 96), F32, F32, F32, seed=8)
    names = ("x", "r", "w", "b")
    leaves = [i[k].requires_grad_(True) for k in names]
    grads = torch.autograd.grad(add_layer_norm(*leaves), leaves, (i["dy"], i["dh"]))
    g = torch.Generator(device=cuda_device).manual_seed(1)
    for k, name in enumerate(names):
        step = torch.randn(leaves[k].shape, generator=g, device=cuda_device)
        sides = []
        for sign in (1.0, -1.0):
            moved = [t.detach() for t in leaves]
            moved[k] = moved[k] + sign * 1e-2 * step
            y, h = add_layer_norm(*moved)
            sides.append(float((y.double() * i["dy"].double()).sum() + (h.double() * i["dh"].double()).sum()))
        difference = (sides[0] - sides[1]) / 2e-2
        gradient = float((grads[k].double() * step.double()).sum())
        assert abs(difference - gradient) <= 2e-3 * max(abs(gradient), float(grads[k].double().norm())), name


def test_large_offset_and_far_mean(cuda_device):
    """A mean far from zero costs its own rounding, not the square's: the variance is taken about it."""
    from isa.kernels.transformer_block import layer_norm

    g = torch.Generator(device=cuda_device).manual_seed(2)
    x = torch.randn(50, 768, generator=g, device=cuda_device) + 1000.0
    w = torch.ones(768, device=cuda_device)
    print("[case] mean of 1000", flush=True)
    close(layer_norm(x, w), layer_norm64(x, w, None, 1e-5)[0], 1000 * 4 * V, "y")  # the mean's error, u 1000, on values of 1


def test_rows_past_32_bit_offsets(cuda_device):
    from isa.kernels.transformer_block import layer_norm

    rows, dim = 2_900_000, 768
    assert rows * dim > 2 ** 31
    print("[case] offsets past 2^31", flush=True)
    x = torch.zeros(rows, dim, dtype=BF16, device=cuda_device)
    x[-5:] = torch.randn(5, dim, device=cuda_device).to(BF16)
    w = torch.ones(dim, dtype=BF16, device=cuda_device)
    y = layer_norm(x, w)
    close(y[-5:], layer_norm64(x[-5:], w, None, 1e-5)[0], UNIT[BF16] + 16 * V, "last rows")


@pytest.mark.parametrize("types", [(F32, F32, F32), (BF16, F32, F32)], ids=str)
def test_bits_repeat_on_any_stream(cuda_device, types):
    from isa.kernels.transformer_block import add_layer_norm

    i = make(cuda_device, (3000, 384), *types)
    leaves = [i[k].requires_grad_(True) for k in ("x", "r", "w", "b")]

    def once():
        y, h = add_layer_norm(*leaves)
        return (y.detach(), h.detach(), *torch.autograd.grad((y, h), leaves, (i["dy"], i["dh"])))

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(first, second))


def test_refusals(cuda_device):
    from isa.kernels.transformer_block import add_layer_norm, layer_norm

    x = torch.zeros(4, 32, device=cuda_device)
    w = torch.ones(32, device=cuda_device)

    def refused(match, f, *args):
        with pytest.raises(RuntimeError, match=match):
            f(*args)

    refused("CUDA", layer_norm, x.cpu(), w)
    refused("must be float32", layer_norm, x.double(), w.double())
    refused("weight must be", layer_norm, x, w.half())
    refused("weight must be", layer_norm, x, w[:16])
    refused("bias", layer_norm, x, w, w[:16])
    refused("one shape", add_layer_norm, x[:2], x, w)
    refused("x must be", add_layer_norm, x, x.half(), w.half())
    refused("last dimension", layer_norm, torch.zeros(2, 16385, device=cuda_device), torch.ones(16385, device=cuda_device))
    refused("eps", layer_norm, x, w, None, -1.0)
