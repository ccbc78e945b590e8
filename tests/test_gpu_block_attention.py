"""window_attention against its formulas in 64 bits.

Tolerances (2-norm of the error over the result's, u the type's unit roundoff): a 16-bit output
carries its own rounding and that of the weights p that its product is taken with, at most u each and
not aligned with one another, so 4 u; a gradient also those of ds and of the output in
delta = do . out, 8 u. In fp32 a weight's relative error is its score's absolute one, some u times
a score of up to about 10 and the D-term sum's length, 64 u; 128 u for gradients.
"""

from __future__ import annotations

import math

import pytest
import torch

from tests.block_helpers import UNIT, attention64, close, visible

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def tolerances(dtype):
    u = UNIT[dtype]
    return (64 * u, 128 * u) if dtype == F32 else (4 * u, 8 * u)


def inputs(dev, b, m, n, h, kv, d, dtype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(*shape, generator=g, device=dev).to(dtype)
            for shape in ((b, m, h, d), (b, n, kv, d), (b, n, kv, d), (b, m, h, d))]


CASES = [
    # batch, queries, keys, heads, kv_heads, head_dim, window, sinks, lengths
    (1, 1, 1, 1, 1, 8, None, 0, None),
    (1, 1, 1, 2, 1, 64, 1, 0, None),
    (2, 1, 65, 4, 2, 64, 16, 3, None),
    (3, 1, 300, 8, 1, 128, 40, 4, [300, 1, 0]),
    (2, 5, 3, 2, 2, 32, None, 0, None),             # more queries than keys: rows that see nothing
    (2, 33, 33, 3, 3, 40, 7, 2, None),
    (1, 64, 64, 2, 2, 64, None, 0, None),
    (1, 65, 129, 2, 1, 64, 64, 64, None),           # window and sinks end with a tile
    (1, 130, 257, 2, 2, 72, 65, 65, None),          # and just past one
    (2, 127, 128, 6, 2, 80, 1, 0, None),            # only the query's own token
    (2, 129, 129, 4, 1, 96, 1000, 5, [129, 60]),
    (3, 200, 200, 3, 1, 128, 50, 300, [200, 0, 77]),  # sinks past the keys; a sequence of none
    (1, 300, 300, 4, 4, 64, 100, 0, None),
    (2, 96, 512, 8, 2, 120, 128, 4, [512, 100]),
    (1, 257, 700, 5, 5, 16, 31, 1, None),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_matches_formulas(cuda_device, case, dtype):
    b, m, n, h, kv, d, window, sinks, lengths = case
    print(f"[case] attention {case} {dtype}", flush=True)
    q, k, v, g = inputs(cuda_device, b, m, n, h, kv, d, dtype, seed=sum(case[:6]))
    from isa.kernels.transformer_block import window_attention

    given = None if lengths is None else torch.tensor(lengths, device=cuda_device, dtype=torch.int32)
    want = attention64(q, k, v, window, sinks, 1.0 / math.sqrt(d), lengths, g)
    for t in (q, k, v):
        t.requires_grad_(True)
    out = window_attention(q, k, v, window=window, sinks=sinks, key_lengths=given)
    got = (out, *torch.autograd.grad(out, (q, k, v), g))
    with torch.no_grad():
        alone = window_attention(q, k, v, window=window, sinks=sinks, key_lengths=given)
    forward, backward = tolerances(dtype)
    for x, w, name in zip(got, want, ("out", "dq", "dk", "dv")):
        assert x.dtype == dtype
        if float(w.abs().max()) < 1e-12:  # a single key: its score has no gradient
            assert float(x.double().abs().max()) <= 64 * backward, name
        else:
            close(x, w, forward if name == "out" else backward, name)
    close(alone, want[0], forward, "without gradients")
    empty = ~visible(b, m, n, window, sinks, lengths).any(2)
    assert torch.count_nonzero(out.detach().cpu()[empty.expand(b, m)]) == 0


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_unseen_slots_are_not_read(cuda_device, dtype):
    """Slots behind a sequence's end and, for a single token, all others that it does not see may hold anything."""
    from isa.kernels.transformer_block import window_attention

    b, n, h, kv, d, window, sinks = 3, 900, 4, 2, 64, 100, 5
    lengths = [900, 333, 70]
    q, k, v, _ = inputs(cuda_device, b, 1, n, h, kv, d, dtype)
    seen = visible(b, 1, n, window, sinks, lengths).any(1).to(cuda_device)
    for t, bad in ((k, math.nan), (v, math.inf)):
        t.masked_fill_(~seen[:, :, None, None], bad)
    print(f"[case] unseen slots {dtype}", flush=True)
    given = torch.tensor(lengths, device=cuda_device)
    out = window_attention(q, k, v, window=window, sinks=sinks, key_lengths=given)
    close(out, attention64(q, k, v, window, sinks, 0.125, lengths)[0], tolerances(dtype)[0], "out")
    # a chunk of tokens: what lies behind the end, in the forward and the backward
    q, k, v, g = inputs(cuda_device, b, 50, n, h, kv, d, dtype, seed=1)
    want = attention64(q, k, v, window, sinks, 0.125, lengths, g)
    for i, length in enumerate(lengths):
        k[i, length:], v[i, length:] = math.nan, -math.inf
    for t in (q, k, v):
        t.requires_grad_(True)
    out = window_attention(q, k, v, window=window, sinks=sinks, key_lengths=given)
    grads = torch.autograd.grad(out, (q, k, v), g)
    for x, w, name in zip((out, *grads), want, ("out", "dq", "dk", "dv")):
        close(x, w, tolerances(dtype)[name != "out"], name)


def test_infinite_scores(cuda_device):
    """Scores far apart: one key takes all, the others' weights vanish; the lowest values of the type stay finite."""
    from isa.kernels.transformer_block import window_attention

    q, k, v, _ = inputs(cuda_device, 1, 70, 70, 2, 2, 64, F32)
    q, k = q * 30.0, k * 30.0
    print("[case] large scores", flush=True)
    out = window_attention(q, k, v)
    close(out, attention64(q, k, v, None, 0, 0.125, None)[0], 2e-4, "out")  # u times scores of some 1000
    k[:, 3] = -1e30  # a finite lowest value, as masks by addition leave it
    assert torch.isfinite(window_attention(q.abs(), k, v)).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_strides(cuda_device, dtype):
    """Views of a joint projection, a longer cache, heads before tokens, broadcast and unaligned operands."""
    from isa.kernels.transformer_block import window_attention

    dev, b, n, h, d = cuda_device, 2, 140, 4, 64
    forward, backward = tolerances(dtype)
    g = torch.Generator(device=dev).manual_seed(5)

    def check(q, k, v, what):
        print(f"[case] strides: {what} {dtype}", flush=True)
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        dout = torch.randn(q.shape, generator=g, device=dev).to(dtype)
        out = window_attention(*leaves, window=50, sinks=2)
        grads = torch.autograd.grad(out, leaves, dout)
        want = attention64(*leaves, 50, 2, 1.0 / math.sqrt(q.shape[3]), None, dout)
        for x, w, name in zip((out, *grads), want, ("out", "dq", "dk", "dv")):
            close(x, w, forward if name == "out" else backward, name)

    joint = torch.randn(b, n, 3, h, d, generator=g, device=dev).to(dtype)
    check(*joint.unbind(2), "joint projection")
    cache = torch.randn(2, b, 2 * n, h, d, generator=g, device=dev).to(dtype)
    check(joint[:, :, 0], cache[0, :, :n], cache[1, :, 7:n + 7], "a longer cache")
    heads_first = torch.randn(3, b, h, n, d, generator=g, device=dev).to(dtype).transpose(2, 3)
    check(*heads_first.unbind(0), "heads before tokens")
    one = torch.randn(b, n, 1, d, generator=g, device=dev).to(dtype)
    check(joint[:, :, 0], one.expand(b, n, h, d), one.expand(b, n, h, d), "broadcast heads")
    odd = torch.randn(b, n, h, d + 3, generator=g, device=dev).to(dtype)[..., 1:d + 1]
    check(odd, odd, odd, "unaligned")
    apart = torch.randn(b, n, h, d, 2, generator=g, device=dev).to(dtype)[..., 0]
    check(apart, apart, apart, "elements apart")
    dev_out = torch.randn(b, h, n, d, generator=g, device=dev).to(dtype).transpose(1, 2)
    leaf = joint[:, :, 0].detach().contiguous().requires_grad_(True)
    out = window_attention(leaf, joint[:, :, 1], joint[:, :, 2], window=50)
    (dq,) = torch.autograd.grad(out, leaf, dev_out)
    close(dq, attention64(leaf, joint[:, :, 1], joint[:, :, 2], 50, 0, 0.125, None, dev_out)[1], backward,
          "gradient with heads before tokens")


def test_shared_heads_and_subsets_of_gradients(cuda_device):
    from isa.kernels.transformer_block import window_attention

    q, k, v, g = inputs(cuda_device, 2, 150, 150, 8, 2, 64, F32)
    want = attention64(q, k, v, 40, 3, 0.125, None, g)
    for wanted in ((0,), (1,), (2,), (0, 2)):
        print(f"[case] gradients of operands {wanted}", flush=True)
        leaves = [t.detach().clone().requires_grad_(i in wanted) for i, t in enumerate((q, k, v))]
        out = window_attention(*leaves, window=40, sinks=3)
        out.backward(g)
        for i, t in enumerate(leaves):
            assert (t.grad is not None) == (i in wanted)
            if i in wanted:
                close(t.grad, want[1 + i], tolerances(F32)[1], f"operand {i}")


def test_gradient_against_differences(cuda_device):
    """The derivative along a random direction, by central differences of the fp32 forward: steps of
    h = 1e-2 leave h^2 of the third derivative and u / h of rounding, some 1e-4 of it each."""
    from isa.kernels.transformer_block import window_attention

    q, k, v, g = inputs(cuda_device, 2, 60, 90, 4, 2, 32, F32, seed=3)
    gen = torch.Generator(device=cuda_device).manual_seed(9)

    def value(q, k, v):
        return float((window_attention(q, k, v, window=20, sinks=2).double() * g.double()).sum())

    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(window_attention(*leaves, window=20, sinks=2), leaves, g)
    for i, name in enumerate("qkv"):
        print(f"[case] differences along {name}", flush=True)
        step = torch.randn((q, k, v)[i].shape, generator=gen, device=cuda_device)
        sides = []
        for sign in (1.0, -1.0):
            moved = [q, k, v]
            moved[i] = moved[i] + sign * 1e-2 * step
            sides.append(value(*moved))
        by_difference = (sides[0] - sides[1]) / 2e-2
        by_gradient = float((grads[i].double() * step.double()).sum())
        spread = float(grads[i].double().norm())  # the standard deviation of such a derivative
        assert abs(by_difference - by_gradient) <= 2e-3 * max(abs(by_gradient), spread), (by_difference, by_gradient)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_bits_repeat_on_any_stream(cuda_device, dtype):
    from isa.kernels.transformer_block import window_attention

    q, k, v, g = inputs(cuda_device, 2, 333, 333, 6, 3, 64, dtype)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def once():
        out = window_attention(*leaves, window=70, sinks=4)
        return (out.detach(), *torch.autograd.grad(out, leaves, g))

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(first, second))


def test_token_of_a_long_cache(cuda_device):
    """Offsets past 2^31 elements: the last tokens of a cache of 2.2 million, of which only what is seen is filled."""
    from isa.kernels.transformer_block import window_attention

    n, h, kv, d, window, sinks = 2_200_000, 8, 8, 128, 200, 4
    assert n * kv * d > 2 ** 31
    print("[case] long cache", flush=True)
    g = torch.Generator(device=cuda_device).manual_seed(2)
    k, v = (torch.empty(1, n, kv, d, dtype=BF16, device=cuda_device) for _ in range(2))
    for t in (k, v):
        t[:, :sinks] = torch.randn(1, sinks, kv, d, generator=g, device=cuda_device).to(BF16)
        t[:, n - window - 3:] = torch.randn(1, window + 3, kv, d, generator=g, device=cuda_device).to(BF16)
    q = torch.randn(1, 3, h, d, generator=g, device=cuda_device).to(BF16)
    out = window_attention(q, k, v, window=window, sinks=sinks)
    short = [torch.cat([t[:, :sinks], t[:, n - window - 3:]], 1) for t in (k, v)]
    want = attention64(q, *short, window, sinks, 1.0 / math.sqrt(d), None)[0]
    close(out, want, tolerances(BF16)[0], "out")


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_tokens_after_a_prompt_match_the_whole(cuda_device, dtype):
    """A prompt, a chunk and single tokens over its cache give what one call over all gives."""
    from isa.kernels.transformer_block import window_attention

    q, k, v, _ = inputs(cuda_device, 2, 260, 260, 4, 2, 64, dtype)
    whole = window_attention(q, k, v, window=90, sinks=4)
    parts = [window_attention(q[:, a:e], k[:, :e], v[:, :e], window=90, sinks=4)
             for a, e in ((0, 150), (150, 257), (257, 258), (258, 259), (259, 260))]
    print(f"[case] prompt, chunk, tokens {dtype}", flush=True)
    close(torch.cat(parts, 1), whole, 2 * tolerances(dtype)[0], "parts")


def test_empty_calls(cuda_device):
    from isa.kernels.transformer_block import window_attention

    def empty(b, m, n):
        q = torch.randn(b, m, 4, 64, device=cuda_device, requires_grad=True)
        k, v = (torch.randn(b, n, 2, 64, device=cuda_device, requires_grad=True) for _ in range(2))
        out = window_attention(q, k, v, window=8)
        assert out.shape == q.shape and torch.count_nonzero(out) == 0
        for t, x in zip(torch.autograd.grad(out, (q, k, v), torch.ones_like(out)), (q, k, v)):
            assert t.shape == x.shape and torch.count_nonzero(t) == 0

    for shape in ((0, 3, 3), (2, 0, 5), (2, 4, 0)):
        print(f"[case] empty {shape}", flush=True)
        empty(*shape)


def test_graph_replays(cuda_device):
    from isa.kernels.transformer_block import window_attention

    q, k, v, g = inputs(cuda_device, 2, 1, 500, 8, 2, 64, BF16)
    lengths = torch.tensor([500, 20], dtype=torch.int32, device=cuda_device)

    def call():
        return window_attention(q, k, v, window=100, sinks=4, key_lengths=lengths)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        print(f"[case] replay {i}", flush=True)
        q.copy_(torch.randn_like(q))
        lengths.copy_(torch.tensor([500 - 100 * i, 20 + i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())


def test_gradients_replay_from_a_graph(cuda_device):
    """A captured forward and backward, replayed on new values between eager runs, give the eager bits."""
    from isa.kernels.transformer_block import window_attention

    q, k, v, g = inputs(cuda_device, 1, 400, 400, 4, 2, 64, BF16)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def call():
        out = window_attention(*leaves, window=100, sinks=4)
        return (out, *torch.autograd.grad(out, leaves, g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for i in range(4):
        print(f"[case] replay {i}", flush=True)
        with torch.no_grad():
            for t in (*leaves, g):
                t.copy_(torch.randn_like(t))
        graph.replay()
        torch.cuda.synchronize()
        for x, w in zip(got, call()):
            assert torch.equal(x, w)


def test_refusals(cuda_device):
    from isa.kernels.transformer_block import window_attention

    q, k, v, _ = inputs(cuda_device, 2, 4, 6, 4, 2, 64, F32)

    def refused(match, *args, **more):
        with pytest.raises(RuntimeError, match=match):
            window_attention(*args, **more)

    refused("CUDA", q.cpu(), k, v)
    refused("must be float32", q.double(), k, v)
    refused("k must be torch.float32", q, k.half(), v)
    refused("head_dim must be", q[..., :12], k[..., :12], v[..., :12])
    wide = torch.zeros(1, 2, 1, 136, device=cuda_device)
    refused("head_dim must be", wide, wide, wide)
    refused("multiple of kv_heads", q[:, :, :3], k, v)
    refused("batch and head_dim", q[:1], k, v)
    refused("got", q, k, v[:, :5])
    refused("window", q, k, v, window=0)
    refused("sinks", q, k, v, sinks=-1)
    refused("scale", q, k, v, scale=0.0)
    refused("scale", q, k, v, scale=math.nan)
    refused("key_lengths", q, k, v, key_lengths=torch.ones(3, dtype=torch.int32, device=cuda_device))
    refused("key_lengths", q, k, v, key_lengths=torch.ones(2, device=cuda_device))
    refused("key_lengths", q, k, v, key_lengths=torch.ones(2, dtype=torch.int32))
    q.requires_grad_(True)
    (dq,) = torch.autograd.grad(window_attention(q, k, v).sum(), q)
    assert not dq.requires_grad
    with pytest.raises(RuntimeError, match="first derivatives only"):
        torch.autograd.grad(window_attention(q, k, v).sum(), q, create_graph=True)
    q.requires_grad_(False)
    # lengths out of range are held to it
    far = window_attention(q, k, v, key_lengths=torch.tensor([99, -5], device=cuda_device))
    close(far, attention64(q, k, v, None, 0, 0.125, [6, 0])[0], tolerances(F32)[0], "lengths held to the keys")


LONG = [
    # the walks over queries are cut: of tiles with sinks, of all tiles, of both, of none but the sinks'
    (1, 1500, 1500, 4, 1, 64, 70, 200, None),
    (1, 1100, 1100, 2, 2, 128, 40, 4, None),
    (1, 700, 700, 3, 1, 96, None, 0, None),
    (2, 900, 1400, 4, 2, 128, 300, 130, [1400, 640]),
    (4, 600, 600, 16, 16, 32, 64, 33, None),
    (1, 40, 3000, 4, 2, 64, 1000, 100, None),       # few rows against many keys: the keys are cut
    (2, 3, 2500, 8, 1, 128, None, 0, [2500, 17]),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("case", LONG, ids=str)
def test_long_walks(cuda_device, case, dtype):
    from isa.kernels.transformer_block import window_attention

    b, m, n, h, kv, d, window, sinks, lengths = case
    print(f"[case] attention {case} {dtype}", flush=True)
    q, k, v, g = inputs(cuda_device, b, m, n, h, kv, d, dtype, seed=sum(case[:6]))
    given = None if lengths is None else torch.tensor(lengths, device=cuda_device, dtype=torch.int32)
    want = attention64(q, k, v, window, sinks, 1.0 / math.sqrt(d), lengths, g)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = window_attention(*leaves, window=window, sinks=sinks, key_lengths=given)
    forward, backward = tolerances(dtype)
    for x, w, name in zip((out, *torch.autograd.grad(out, leaves, g)), want, ("out", "dq", "dk", "dv")):
        close(x, w, forward if name == "out" else backward, name)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("scale", [2.0 ** -17, 2.0 ** 12])
def test_gradients_of_any_size(cuda_device, dtype, scale):
    """Gradients of a mean loss are small, those of a scaled one large: the result scales with them, to
    what its type holds (in fp16 2^-25 is half its smallest number)."""
    from isa.kernels.transformer_block import window_attention

    print(f"[case] gradients of {scale} {dtype}", flush=True)
    for m, n, window, sinks in ((200, 200, 64, 3), (900, 900, 100, 4)):
        q, k, v, g = inputs(cuda_device, 1, m, n, 4, 2, 64, dtype, seed=11)
        g = (g.float() * scale).to(dtype)
        want = attention64(q, k, v, window, sinks, 0.125, None, g)[1:]
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        out = window_attention(*leaves, window=window, sinks=sinks)
        for x, w, name in zip(torch.autograd.grad(out, leaves, g), want, ("dq", "dk", "dv")):
            floor = 2.0 ** -25 * math.sqrt(w.numel()) / float(w.norm()) if dtype == F16 else 0.0
            close(x, w, tolerances(dtype)[1] + floor, name)
        # keys and values alone, whose kernel takes the rows' sums from elsewhere
        k2, v2 = (t.detach().clone().requires_grad_(True) for t in (k, v))
        for x, w, name in zip(torch.autograd.grad(window_attention(q.detach(), k2, v2, window=window, sinks=sinks), (k2, v2), g),
                              want[1:], ("dk alone", "dv alone")):
            floor = 2.0 ** -25 * math.sqrt(w.numel()) / float(w.norm()) if dtype == F16 else 0.0
            close(x, w, tolerances(dtype)[1] + floor, name)
