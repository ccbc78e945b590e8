"""Embedding lookup and the tables' gradients against their formulas in 64 bits.

Tolerances, element by element (u of the type, v = 2^-24): y is one fp32 sum, rounded once: (u + 2 v) |y|. A gradient's
sum of L terms is made in at most `depth` additions one after the other, each off by v of at most the sum S of the
terms' sizes, then scaled and rounded: u |g| + v (depth + 2) S. 16 bits: what is below the smallest number of fp16,
half of 2^-24, is lost besides.
"""

from __future__ import annotations

import math

import pytest
import torch

from tests.block_helpers import UNIT
from tests.train_helpers import embedding64

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
V = UNIT[F32]


def within(got, want, bound, what):
    g = got.detach().double().cpu()
    assert g.shape == want.shape, (what, g.shape, want.shape)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(g), nan), what
    over = ((g - want).abs() - bound).masked_fill(nan, -1.0)
    assert not over.numel() or float(over.max()) <= 0.0, (what, float(over.max()), int((over > 0).sum()))


def depth(tokens):
    """Additions one after the other. Up to 2048 tokens: those of one of a block's 16 to 128 groups, then of the groups;
    else a tile's, then of every eighth tile, then of eight waves."""
    if tokens <= 2048:
        return -(-tokens // 16) + 128
    tile = max(16, -(-tokens // 2048))
    return tile + -(-tokens // tile // 8) + 9


def check(dev, ids, weight, scale=1.0, positions=None, position_weight=None, padding=None, seed=0):
    from isa.kernels.transformer_block import embedding

    dtype, dim = weight.dtype, weight.shape[1]
    how = {"scale": scale, "positions": positions, "position_weight": position_weight, "padding_index": padding}
    g = torch.Generator(device=dev).manual_seed(seed)
    dy = torch.randn(*ids.shape, dim, generator=g, device=dev).to(dtype)
    leaves = [weight.detach().requires_grad_(True)]
    if position_weight is not None:
        leaves.append(position_weight.detach().requires_grad_(True))
        how["position_weight"] = leaves[1]
    y = embedding(ids, leaves[0], **how)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        assert torch.equal(embedding(ids, weight, **how), y) or bool(torch.isnan(y).any())
    flat = ids.reshape(-1)
    at = None
    if position_weight is not None:
        at = positions
        if at is None:
            at = torch.arange(ids.shape[-1], device=dev) if ids.dim() else torch.zeros_like(ids)
        at = at.expand(ids.shape).reshape(-1)
    want = embedding64(flat, weight, scale, at, position_weight, padding, dy)
    sizes = embedding64(flat, weight, abs(scale), at, position_weight, padding, dy.abs())
    tiny = 2.0 ** -25 if dtype == F16 else 0.0
    within(y.reshape(-1, dim), want[0], (UNIT[dtype] + 2 * V) * want[0].abs() + tiny, "y")
    for got, w, s, name in zip(grads, want[1:], sizes[1:], ("dweight", "dposition_weight")):
        assert got.dtype == dtype
        within(got, w, UNIT[dtype] * w.abs() + V * (depth(flat.numel()) + 2) * s + tiny, name)
    again = torch.autograd.grad(embedding(ids, leaves[0], **how), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    return y, grads


def make(dev, shape, vocab, dim, dtype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    n = math.prod(shape)
    u = torch.rand(n, generator=g, device=dev, dtype=torch.float64)
    ids = (torch.pow(vocab + 1.0, u) - 1.0).long().clamp_(0, vocab - 1).view(shape)
    return ids, torch.randn(vocab, dim, generator=g, device=dev).to(dtype)


# (ids' shape, vocab, dim): single ones, a table of one row, rows of every remainder, several ranges of the sort and more
# than 512 x 256 rows, lists of several tiles, rows wider than a block
SIZES = [((1,), 1, 1), ((5,), 3, 2), ((2, 7), 11, 3), ((63,), 64, 8), ((64,), 7, 9), ((65,), 7, 20), ((3, 100), 1000, 33),
         ((1000,), 5, 40), ((4, 257), 257, 390), ((999,), 5003, 129), ((2, 1024), 50304, 64), ((777,), 140001, 17),
         ((8, 513), 300, 1028), ((300,), 40, 5000), ((20000,), 2, 24), ((1,), 50304, 768), ((3000,), 513, 7)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_matches_formulas(cuda_device, size, dtype):
    print(f"[case] embedding {size} {dtype}", flush=True)
    ids, w = make(cuda_device, *size, dtype, seed=sum(size[0]))
    check(cuda_device, ids, w)
    check(cuda_device, ids, w, scale=-3.3, padding=0)
    n = ids.shape[-1]
    g = torch.Generator(device=cuda_device).manual_seed(1)
    for rows in (n, n + 5):
        p = torch.randn(rows, w.shape[1], generator=g, device=cuda_device).to(dtype)
        check(cuda_device, ids, w, 2.0, None, p)
        at = torch.randint(0, rows, ids.shape, generator=g, device=cuda_device)
        check(cuda_device, ids.int(), w, 0.5, at, p, seed=3)
    check(cuda_device, ids, w, 1.0, at[..., :1].int(), p)  # one place for all


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_ids_and_positions_outside_their_tables(cuda_device, dtype):
    """NaN rows, and no part in that table's gradient (in the other one's they have)."""
    ids, w = make(cuda_device, (6, 50), 31, 24, dtype)
    ids[0, :7] = torch.tensor([-1, 31, 2 ** 40, -(2 ** 62), 30, 0, 2 ** 31], device=cuda_device)
    p = torch.randn(60, 24, device=cuda_device).to(dtype)
    at = torch.randint(0, 60, ids.shape, device=cuda_device)
    at[1, :4] = torch.tensor([-1, 60, 2 ** 33, -(2 ** 60)], device=cuda_device)
    y, _ = check(cuda_device, ids, w)
    assert int(torch.isnan(y[0, :, 0]).sum()) == 5
    check(cuda_device, ids, w, 1.5, at, p, padding=2)
    check(cuda_device, torch.full((5, 9), 31, device=cuda_device), w, 1.0, None, p)  # none inside
    check(cuda_device, torch.full((700,), 3, device=cuda_device), w, padding=3)  # none but padding


def test_one_token_again_and_again(cuda_device):
    """A list over many tiles, whole and cut ones, beside short ones; and a table where every second row is long."""
    w = torch.randn(10, 40, device=cuda_device)
    for n in (64, 65, 128, 1000, 131073, 200001):
        print(f"[case] {n} times one token", flush=True)
        check(cuda_device, torch.full((n,), 4, device=cuda_device), w)
        check(cuda_device, torch.cat([torch.full((n,), 4), torch.arange(10), torch.full((77,), 5)]).to(cuda_device), w, padding=9)
    check(cuda_device, torch.arange(5, device=cuda_device).repeat(300) * 2, w)
    check(cuda_device, torch.arange(5, device=cuda_device).repeat(64) * 2, w)
    check(cuda_device, torch.arange(5, device=cuda_device).repeat_interleave(65) * 2, w)
    p = torch.randn(3, 40, device=cuda_device)
    for times in (200, 5000):  # positions that many tokens share
        check(cuda_device, torch.zeros(times, 2, dtype=torch.int64, device=cuda_device), w, 1.0, None, p)
    for dim in (3, 64, 700, 1500):  # long rows of few tokens, by every width of a group
        w = torch.randn(60, dim, device=cuda_device)
        for dtype in (F32, BF16):
            ids = torch.cat([torch.full((900,), 59), torch.arange(60), torch.full((40,), 3), torch.full((17,), 4)]).to(cuda_device)
            check(cuda_device, ids, w.to(dtype), 0.5)


def test_views_and_empty_ones(cuda_device):
    from isa.kernels.transformer_block import embedding

    whole = torch.randn(50, 37, device=cuda_device)
    ids = torch.randint(0, 25, (8, 12), device=cuda_device)
    for name, w in (("rows apart", whole[:, 3:36]), ("every second row", whole[::2]), ("elements apart", whole[:, ::2]),
                    ("a transposed table", whole.t().contiguous().t()), ("one row for all", whole[:1].expand(50, 37))):
        print(f"[case] {name}", flush=True)
        check(cuda_device, ids, w, 1.0, None, w)
    check(cuda_device, ids.t(), whole)
    check(cuda_device, ids[::2, 1::3], whole, 1.0, ids[:1, 1::3], whole)
    check(cuda_device, ids[0, 0], whole, 1.0, None, whole)  # no dimension
    y, (g,) = check(cuda_device, ids, whole[:0])  # a table without rows
    assert torch.isnan(y).all() and g.shape == (0, 37)
    for shape in ((0,), (3, 0), (0, 5)):
        print(f"[case] empty {shape}", flush=True)
        none = torch.zeros(shape, dtype=torch.int64, device=cuda_device)
        leaf = whole.clone().requires_grad_(True)
        y = embedding(none, leaf, position_weight=leaf)
        assert y.shape == (*shape, 37)
        (g,) = torch.autograd.grad(y, leaf, torch.zeros_like(y))
        assert g.shape == whole.shape and torch.count_nonzero(g) == 0
    # a gradient that is spread out, and one that came as a view
    leaf = whole.clone().requires_grad_(True)
    (a,) = torch.autograd.grad(embedding(ids, leaf).sum(), leaf)
    (b,) = torch.autograd.grad(embedding(ids, leaf), leaf, torch.ones(8, 12, 37, device=cuda_device))
    assert torch.equal(a, b)
    up = torch.randn(12, 8, 37, device=cuda_device).transpose(0, 1)
    (a,) = torch.autograd.grad(embedding(ids, leaf), leaf, up)
    (b,) = torch.autograd.grad(embedding(ids, leaf), leaf, up.contiguous())
    assert torch.equal(a, b)


def test_only_one_table_learns(cuda_device):
    from isa.kernels.transformer_block import embedding

    ids, w = make(cuda_device, (3, 20), 50, 16, F32)
    p = torch.randn(20, 16, device=cuda_device)
    dy = torch.randn(3, 20, 16, device=cuda_device)
    both = [w.clone().requires_grad_(True), p.clone().requires_grad_(True)]
    want = torch.autograd.grad(embedding(ids, both[0], position_weight=both[1]), both, dy)
    for i in range(2):
        leaves = [w.clone(), p.clone()]
        leaves[i].requires_grad_(True)
        (got,) = torch.autograd.grad(embedding(ids, leaves[0], position_weight=leaves[1]), leaves[i], dy)
        assert torch.equal(got, want[i])


def test_gradient_against_differences(cuda_device):
    """sum(y c) is linear in the tables: differences over a step of 1 are exact up to fp32 sums of some 400 terms."""
    from isa.kernels.transformer_block import embedding

    ids, w = make(cuda_device, (4, 9), 12, 8, F32, seed=5)
    p, c = torch.randn(9, 8, device=cuda_device), torch.randn(4, 9, 8, device=cuda_device)
    leaves = [w.requires_grad_(True), p.requires_grad_(True)]
    f = lambda a, b: (embedding(ids, a, scale=1.5, position_weight=b).double() * c.double()).sum()  # noqa: E731
    grads = torch.autograd.grad(embedding(ids, *leaves[:1], scale=1.5, position_weight=leaves[1]), leaves, c)
    with torch.no_grad():
        for i, (leaf, g) in enumerate(zip(leaves, grads)):
            for at in ((0, 0), (3, 5), (8, 7)):
                moved = [t.clone() for t in leaves]
                moved[i][at] += 1.0
                diff = float(f(*moved)) - float(f(*leaves))
                assert abs(diff - float(g[at])) <= 400 * V * 8 * max(1.0, float(g.abs().max())), (i, at)


@pytest.mark.parametrize("size", [(1500, 50304, 200, F32), (3000, 50304, 512, F32), (70000, 40000, 1024, BF16), (40, 90000, 390, BF16)],
                         ids=str)
def test_large_tables_and_results(cuda_device, size):
    """Tables and results past the sizes from which tiles are made of few tokens and writes go past the caches; the 64-bit
    sums are made on the GPU."""
    from isa.kernels.transformer_block import embedding

    tokens, vocab, dim, dtype = size
    print(f"[case] {size}", flush=True)
    ids, w = make(cuda_device, (tokens,), vocab, dim, dtype, seed=7)
    ids[: tokens // 2] = torch.where(torch.rand(tokens // 2, device=cuda_device) < 0.5, vocab - 1, ids[: tokens // 2])
    g = torch.Generator(device=cuda_device).manual_seed(8)
    dy = torch.randn(tokens, dim, generator=g, device=cuda_device).to(dtype)
    w.requires_grad_(True)
    y = embedding(ids, w)
    assert torch.equal(y, w.detach()[ids])
    (dw,) = torch.autograd.grad(y, w, dy)
    want = torch.zeros(vocab, dim, dtype=torch.float64, device=cuda_device).index_add_(0, ids, dy.double())
    sizes = torch.zeros_like(want).index_add_(0, ids, dy.double().abs())
    over = (dw.double() - want).abs() - UNIT[dtype] * want.abs() - V * (depth(tokens) + 2) * sizes
    assert float(over.max()) <= 0.0
