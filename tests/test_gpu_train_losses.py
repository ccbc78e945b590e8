"""The policy loss and the preference loss against their formulas in 64 bits.

Tolerances (u of the result's type, v = 2^-24): l is a difference of numbers up to some 20: 64 v of the largest one;
so is what the exponent of a ratio is made of, and a ratio is off by as much relative to itself. A gradient is a
softmax (20 v and some) times a slope (64 v of the largest number in its exponent) and one rounding.
A preference's margin is a sum in 64 bits of a sequence's l, each off by 64 v of numbers up to 20.
"""

from __future__ import annotations

import math

import pytest
import torch

from tests.block_helpers import UNIT, close
from tests.train_helpers import policy64, preference64

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
V = UNIT[F32]
# rows of 1 to 16 pieces of 16 bytes for each thread of blocks of 256, 512 and 1024, and more
SIZES = [(1, 1), (3, 2), (5, 100), (7, 1023), (4, 4096), (9, 5003), (4, 7001), (3, 9000), (5, 16384), (4, 20001), (3, 28672),
         (4, 36000), (3, 50304), (2, 50305), (2, 65536), (2, 150001), (300, 257)]


def make(dev, rows, vocab, dtype, seed=0, low=0.2, high=0.2):
    """Logits, actions, old, advantages, ref; every third row ignored; no ratio next to a bound."""
    g = torch.Generator(device=dev).manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g, device=dev) * 3.0).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device=dev)
    now = torch.log_softmax(x.double(), -1).gather(1, t[:, None])[:, 0]
    d = torch.randn(rows, generator=g, device=dev).double() * 0.3
    for border in (math.log(1.0 - low) if low < 1.0 else -99.0, math.log(1.0 + high)):
        d = torch.where((d - border).abs() < 1e-3, d + 3e-3, d)
    a = torch.randn(rows, generator=g, device=dev)
    ref = now - torch.randn(rows, generator=g, device=dev) * 0.5
    if rows > 2:
        t[1::3] = -100
    return x, t, (now - d).float(), a, ref.float()


def grads_close(got, want, dtype, extra, what):
    """A 16-bit gradient also loses what is below its type's smallest number."""
    norm = float(want.norm())
    if norm == 0.0:
        assert torch.count_nonzero(got) == 0
        return
    floor = (2.0 ** -25 if dtype == F16 else 0.0) * math.sqrt(want.numel()) / norm
    close(got, want, UNIT[dtype] + extra + floor, what)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_policy_matches_formulas(cuda_device, size, dtype):
    from isa.kernels.transformer_block import policy_loss, policy_loss_with_grad

    for kl, clip in ((0.0, 0.2), (0.1, (0.1, 0.3)), (0.5, None)):
        print(f"[case] policy {size} {dtype} kl {kl} clip {clip}", flush=True)
        low, high = (1.0, math.inf) if clip is None else clip if isinstance(clip, tuple) else (clip, clip)
        x, t, old, a, ref = make(cuda_device, *size, dtype, sum(size), low, high if clip else 0.2)
        row, grad, l = policy64(x, t, old, a, ref, low, high, kl, -100)
        count = int((t != -100).sum())
        # the largest number that l and an exponent are made of, and a slope's size in both parts
        top = max(1.0, float(x.abs().max()), float(l.abs().max()))
        off = 64 * V * top
        parts = (1.0 + kl) * max(1.0, float(a.abs().max())) * math.exp(3.0)
        how = {"ref_logp": ref if kl else None, "kl": kl, "clip": clip}
        for reduction, factor, want in (("mean", 1.0 / count, row.sum() / count), ("sum", 1.0, row.sum()), ("none", 1.0, row)):
            leaf = x.detach().requires_grad_(True)
            loss, logp = policy_loss(leaf, t, old, a, reduction=reduction, **how)
            assert loss.dtype == logp.dtype == F32 and not logp.requires_grad
            assert float((logp.double().cpu() - l).abs().max()) <= off
            many = size[0] if reduction == "sum" else 1
            assert float((loss.double().cpu() - want).abs().max()) <= off * parts * many, reduction
            (dx,) = torch.autograd.grad(loss, leaf, torch.full_like(loss, 0.5))
            assert dx.dtype == dtype
            grads_close(dx, grad * 0.5 * factor, dtype, off * 4, reduction)
            with torch.no_grad():
                again = policy_loss(x, t, old, a, reduction=reduction, **how)
                assert torch.equal(again[0], loss) and torch.equal(again[1], logp)
        loss, dx, logp2 = policy_loss_with_grad(x, t, old, a, grad_scale=8.0, **how)
        # (a row's exponentials are summed in another order than without the gradient)
        assert abs(float(loss) - float(row.sum() / count)) <= off * parts
        assert float((logp2.double().cpu() - l).abs().max()) <= off
        grads_close(dx, grad * (8.0 / count), dtype, off * 4, "one pass")
        assert torch.count_nonzero(dx[t == -100]) == 0


def test_policy_of_sequences_and_views(cuda_device):
    from isa.kernels.transformer_block import cross_entropy, policy_loss, policy_loss_with_grad

    for dtype in (F32, BF16):
        x, t, old, a, ref = make(cuda_device, 24, 1031, dtype, 3)
        t = t.clamp(max=499)
        whole = {"kl": 0.1}
        for k, cut in enumerate((lambda z: z[:, :1000], lambda z: z[:, 1:1002], lambda z: z[:, ::2], lambda z: z[::2, 5:505],
                                 lambda z: z.view(4, 6, 1031), lambda z: z.view(4, 6, 1031)[:, :-1])):
            print(f"[case] view {k} {dtype}", flush=True)
            y = cut(x)
            small = [z[::2] if k == 3 else z.view(4, 6) if k == 4 else z.view(4, 6)[:, :-1] if k == 5 else z for z in (t, old, a, ref)]
            one = policy_loss_with_grad(y, *small[:3], ref_logp=small[3], **whole)
            two = policy_loss_with_grad(y.contiguous().clone(), *(z.contiguous() for z in small[:3]), ref_logp=small[3].contiguous(), **whole)
            assert one[1].shape == y.shape and one[2].shape == small[0].shape
            assert abs(float(one[0]) - float(two[0])) <= 1e-5 * max(1.0, abs(float(two[0])))
            close(one[1], two[1], 2 * UNIT[dtype] + 256 * V, "gradient")
            leaf = y.detach().requires_grad_(True)
            loss, logp = policy_loss(leaf, *small[:3], ref_logp=small[3], **whole)
            close(torch.autograd.grad(loss, leaf)[0], two[1], 2 * UNIT[dtype] + 256 * V, "autograd")
            nll = cross_entropy(y, small[0], reduction="none")
            close(logp, -nll, 64 * V, "logp")
        # an advantage a sequence, spread over its tokens
        spread = a[:4, None].expand(4, 6)
        got = policy_loss_with_grad(x.view(4, 6, -1), t.view(4, 6), old.view(4, 6), spread)
        want = policy_loss_with_grad(x.view(4, 6, -1), t.view(4, 6), old.view(4, 6), spread.contiguous())
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_policy_bounds(cuda_device):
    """Past a bound on the side that the minimum takes no gradient passes; at ratio 1 all of it does; an advantage of 0
    gives none; infinities and actions outside the vocabulary."""
    from isa.kernels.transformer_block import policy_loss, policy_loss_with_grad

    x = torch.randn(8, 50, device=cuda_device)
    t = torch.arange(8, device=cuda_device)
    now = torch.log_softmax(x.double(), -1).gather(1, t[:, None])[:, 0]
    old = (now - torch.tensor([0.5, 0.5, -0.5, -0.5, 0.0, 0.0, 0.5, -0.5], device=cuda_device)).float()
    a = torch.tensor([1.0, -1.0, 1.0, -1.0, 2.0, -2.0, 0.0, 0.0], device=cuda_device)
    loss, dx, _ = policy_loss_with_grad(x, t, old, a)
    assert [bool(r.any()) for r in dx] == [False, True, True, False, True, True, False, False]
    want = policy64(x, t, old, a, None, 0.2, 0.2, 0.0, -100)
    close(dx, want[1] / 8, 256 * V, "gradient")
    for bad in (-1, 50, 2 ** 40):
        u = t.clone()
        u[3] = bad
        loss, dx, logp = policy_loss_with_grad(x, u, old, a)
        assert math.isnan(float(loss)) and torch.isnan(dx[3]).all() and torch.isnan(logp[3])
        rest = [i for i in range(8) if i != 3]
        assert torch.isfinite(dx[rest]).all() and torch.isfinite(logp[rest]).all()
    # a NaN in what is held fixed stays in its row
    for name in ("old", "a", "ref"):
        args = {"old": old.clone(), "a": a.clone(), "ref": old.clone()}
        args[name][2] = math.nan
        rows, _ = policy_loss(x, t, args["old"], args["a"], ref_logp=args["ref"], kl=0.1, reduction="none")
        assert torch.equal(torch.isnan(rows), torch.arange(8, device=cuda_device) == 2), name
    # logits without a part: what is masked keeps a gradient of 0
    y = x.clone()
    y[:, 20:] = -math.inf
    old = (torch.log_softmax(y.double(), -1).gather(1, t[:, None])[:, 0]).float()
    _, dx, _ = policy_loss_with_grad(y, t, old, a)
    assert torch.isfinite(dx).all() and torch.count_nonzero(dx[:, 20:]) == 0
    # nothing that counts, and no rows
    none = torch.full_like(t, -100)
    loss, dx, logp = policy_loss_with_grad(x, none, old, a)
    assert math.isnan(float(loss)) and torch.count_nonzero(dx) == 0 and torch.count_nonzero(logp) == 0
    assert float(policy_loss(x, none, old, a, reduction="sum")[0]) == 0.0
    e = [z[:0] for z in (x, t, old, a)]
    assert policy_loss(*e, reduction="none")[0].shape == (0,) and float(policy_loss(*e, reduction="sum")[0]) == 0.0
    assert policy_loss_with_grad(*e)[1].shape == (0, 50)


def test_policy_gradient_against_differences(cuda_device):
    """Central differences of the loss in 64 bits, whose formula the kernel's loss is held to above."""
    from isa.kernels.transformer_block import policy_loss_with_grad

    x, t, old, a, ref = make(cuda_device, 6, 11, F32, 9)
    _, dx, _ = policy_loss_with_grad(x, t, old, a, ref_logp=ref, kl=0.3)
    f = lambda z: float(policy64(z, t, old, a, ref, 0.2, 0.2, 0.3, -100)[0].sum()) / int((t != -100).sum())  # noqa: E731
    for r, c in ((0, 3), (2, 10), (3, int(t[3])), (5, 0)):
        step = torch.zeros_like(x, dtype=torch.float64)
        step[r, c] = 1e-5
        diff = (f(x.double() + step) - f(x.double() - step)) / 2e-5
        assert abs(diff - float(dx[r, c])) <= 1e-5 * max(1.0, abs(diff)), (r, c, diff, float(dx[r, c]))


def pairs(dev, n, tokens, vocab, dtype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = (torch.randn(2 * n, tokens, vocab, generator=g, device=dev) * 2.0).to(dtype)
    t = torch.randint(0, vocab, (2 * n, tokens), generator=g, device=dev)
    keep = torch.rand(2 * n, tokens, generator=g, device=dev) < 0.7
    if n > 1:
        keep[1] = False  # a sequence without a token that counts
    taken = (torch.log_softmax(x.double(), -1).gather(2, t[..., None])[..., 0] * keep).sum(1)
    return x, t.masked_fill(~keep, -100), (taken + torch.randn(2 * n, generator=g, device=dev).double() * 3.0).float()


PAIRS = [(1, 1, 1), (1, 1, 2), (2, 3, 100), (3, 17, 1023), (2, 300, 257), (1, 5, 5003), (2, 2, 9000), (1, 3, 20001), (2, 2, 50304), (1, 1, 150001), (33, 4, 40),
         (1, 1500, 33)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("size", PAIRS, ids=str)
def test_preference_matches_formulas(cuda_device, size, dtype):
    from isa.kernels.transformer_block import preference_loss, preference_loss_with_grad

    n, tokens, vocab = size
    for beta in (0.1, 1.0):
        print(f"[case] preference {size} {dtype} beta {beta}", flush=True)
        x, t, ref = pairs(cuda_device, *size, dtype, sum(size))
        rows, grad, total = preference64(x, t, ref, beta, -100)
        # l's: the statistics' rounding is shared by no two rows: their errors add up, at worst all of them
        off = 64 * V * 20 * (math.sqrt(tokens) + 1)
        for reduction, factor, want in (("mean", 1.0 / n, rows.mean()), ("sum", 1.0, rows.sum()), ("none", 1.0, rows)):
            leaf = x.detach().requires_grad_(True)
            loss, logp = preference_loss(leaf, t, ref, beta=beta, reduction=reduction)
            assert loss.dtype == logp.dtype == F32 and not logp.requires_grad and logp.shape == (2 * n,)
            assert float(((logp.double().cpu() - total).abs() - V * total.abs()).max()) <= off
            many = n if reduction == "sum" else 1
            assert float(((loss.double().cpu() - want).abs() - 2 * V * want.abs()).max()) <= 2 * beta * off * many, reduction
            (dx,) = torch.autograd.grad(loss, leaf, torch.full_like(loss, 0.5))
            assert dx.dtype == dtype
            grads_close(dx, grad * 0.5 * factor, dtype, 2 * beta * off + 64 * V, reduction)
            with torch.no_grad():
                again = preference_loss(x, t, ref, beta=beta, reduction=reduction)
                assert torch.equal(again[0], loss) and torch.equal(again[1], logp)
        loss, dx, logp2 = preference_loss_with_grad(x, t, ref, beta=beta, grad_scale=4.0)
        assert abs(float(loss) - float(rows.mean())) <= 2 * beta * off + 2 * V * float(rows.mean()) and torch.equal(logp, logp2)
        grads_close(dx, grad * (4.0 / n), dtype, 2 * beta * off + 64 * V, "with grad")
        assert torch.count_nonzero(dx[t == -100]) == 0


def test_preference_edges(cuda_device):
    from isa.kernels.transformer_block import preference_loss, preference_loss_with_grad

    x, t, ref = pairs(cuda_device, 2, 5, 40, F32)
    # each pair's own gradient
    leaf = x.detach().requires_grad_(True)
    rows, _ = preference_loss(leaf, t, ref, reduction="none")
    (dx,) = torch.autograd.grad(rows[1], leaf)
    assert torch.count_nonzero(dx[0]) == 0 and torch.count_nonzero(dx[2]) == 0 and dx[3].any()
    # margins far out on either side: a loss as large as the margin, or 0, without infinities
    for by, want in ((1e4, 1e4), (-1e4, 0.0)):
        far = ref + torch.tensor([by, by, 0.0, 0.0], device=cuda_device)
        loss, dx, _ = preference_loss_with_grad(x, t, far, beta=1.0)
        assert abs(float(loss) - want) <= 0.01 * 1e4 and torch.isfinite(dx).all()
    # a target outside the vocabulary makes its pair NaN and no other
    for bad in (-1, 40, 2 ** 40):
        u = t.clone()
        u[2, 3] = bad
        rows, logp = preference_loss(x, u, ref, reduction="none")
        assert math.isnan(float(rows[0])) and math.isfinite(float(rows[1])) and math.isnan(float(logp[2]))
        _, dx, _ = preference_loss_with_grad(x, u, ref)
        assert torch.isfinite(dx[1]).all() and torch.isfinite(dx[3]).all() and torch.isnan(dx[2, 3]).all()
    # views: more columns than classes, sequences apart, tokens apart
    wide = torch.randn(8, 9, 64, device=cuda_device)
    for k, y in enumerate((wide[:, :, :50], wide[::2], wide[:, ::2], wide.transpose(0, 1)[:8])):
        print(f"[case] view {k}", flush=True)
        u = torch.randint(0, 40, y.shape[:2], device=cuda_device)
        z = torch.randn(y.shape[0], device=cuda_device)
        a, b = preference_loss_with_grad(y, u, z), preference_loss_with_grad(y.contiguous(), u, z)
        for p, q in zip(a, b):
            torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-7)
    # no tokens, no pairs
    loss, dx, logp = preference_loss_with_grad(x[:, :0], t[:, :0], torch.zeros(4, device=cuda_device))
    assert abs(float(loss) - math.log(2.0)) <= 1e-6 and dx.shape == (4, 0, 40) and torch.count_nonzero(logp) == 0
    assert math.isnan(float(preference_loss(x[:0], t[:0], ref[:0])[0]))
    assert float(preference_loss(x[:0], t[:0], ref[:0], reduction="sum")[0]) == 0.0
    assert preference_loss(x[:0], t[:0], ref[:0], reduction="none")[0].shape == (0,)


@pytest.mark.parametrize("vocab", [25000, 25001], ids=str)
def test_large_gradients(cuda_device, vocab):
    """Gradients large enough to be written past the caches are those of a part of the rows, bit by bit."""
    from isa.kernels.transformer_block import policy_loss, policy_loss_with_grad, preference_loss

    x, t, old, a, _ = make(cuda_device, 3000, vocab, BF16, 4)
    assert x.numel() * 2 >= 2 ** 27
    t[400:] = -100
    many = x.detach().requires_grad_(True)
    few = x[:400].detach().requires_grad_(True)
    (dx,) = torch.autograd.grad(policy_loss(many, t, old, a, reduction="sum")[0], many)
    (part,) = torch.autograd.grad(policy_loss(few, t[:400], old[:400], a[:400], reduction="sum")[0], few)
    assert torch.equal(dx[:400], part) and part.any() and torch.count_nonzero(dx[400:]) == 0
    count = float((t[:400] != -100).sum())
    _, dx, _ = policy_loss_with_grad(x, t, old, a, grad_scale=count)
    _, part, _ = policy_loss_with_grad(x[:400], t[:400], old[:400], a[:400], grad_scale=count)
    assert torch.equal(dx[:400], part) and part.any() and torch.count_nonzero(dx[400:]) == 0
    # one chosen sequence of 1500 tokens, of which 400 count, against the same cut behind them
    u = t.view(2, 1500)
    (dx,) = torch.autograd.grad(preference_loss(many.view(2, 1500, vocab), u, old[:2], reduction="sum")[0], many)
    cut = x.view(2, 1500, vocab)[:, :400].contiguous().requires_grad_(True)
    (part,) = torch.autograd.grad(preference_loss(cut, u[:, :400].contiguous(), old[:2], reduction="sum")[0], cut)
    assert torch.equal(dx.view(2, 1500, vocab)[:, :400], part) and part.any()
    assert torch.count_nonzero(dx.view(2, 1500, vocab)[:, 400:]) == 0
