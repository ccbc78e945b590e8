"""How near attention's results come to 64-bit ones rounded once to their type, on inputs where that takes care:
sinks that hold most of a row's weight, rows with one weight near 1, scores far from zero.

Tolerances are ratios of 2-norm errors, the kernel's over that of the 64-bit result rounded once. They are
bounds between two emulations in 64 bits (300 tokens, window 64, 4 sinks, 4 heads on 2 of 64). One has all
roundings of the kernels (p and ds to 16 bits, sinks' in two parts, delta with what out's rounding left):
ratios 1.2 to 1.5 for plain inputs, dq 1.1 and dk and dv to 1.6 with strong sinks, dq and dk 1.6 with
weights near 1. The other is without the second part of sinks' p and ds (dq 1.63 with strong sinks), or
without what out's rounding left (dq 1.72 with strong sinks; dq and dk 8 and more with weights near 1), or
has lse of the rounded weights' sum (dq 2.0 with weights near 1).
"""

from __future__ import annotations

import pytest
import torch

from tests.block_helpers import UNIT, attention64, close, off

pytestmark = pytest.mark.gpu

B, N, H, KV, D, WINDOW, SINKS = 1, 300, 4, 2, 64, 64, 4
LIMITS = {"plain": (1.6, 1.7, 1.7, 1.7), "sinks": (1.3, 1.35, 1.8, 1.8), "one": (1.3, 2.0, 2.0, 1.6)}


def inputs(dev, kind, dtype):
    g = torch.Generator().manual_seed(0)
    q, k, v, dout = (torch.randn(B, N, heads, D, generator=g) for heads in (H, KV, KV, H))
    if kind == "sinks":  # first tokens draw more attention than their content explains
        s = torch.randn(D, generator=g) * 0.5
        q += s
        k[:, :SINKS] += 2.0 * s
    if kind == "one":  # each query points at its own key
        q = q * 0.1 + k.repeat_interleave(H // KV, 2)
    return [t.to(dtype).to(dev) for t in (q, k, v, dout)]


def run(q, k, v, dout, **how):
    from isa.kernels.transformer_block import window_attention

    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = window_attention(*leaves, **how)
    return (out.detach(), *torch.autograd.grad(out, leaves, dout))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("kind", sorted(LIMITS))
@pytest.mark.parametrize("scale", [None, 0.11])
def test_16_bit_results_against_one_rounding(cuda_device, kind, dtype, scale):
    print(f"[case] {kind} {dtype} scale {scale}", flush=True)
    i = inputs(cuda_device, kind, dtype)
    want = attention64(*i[:3], WINDOW, SINKS, scale or 0.125, None, i[3])
    got = run(*i[:3], i[3], window=WINDOW, sinks=SINKS, scale=scale)
    for x, w, limit, name in zip(got, want, LIMITS[kind], ("out", "dq", "dk", "dv")):
        once = off(w.to(dtype), w)[0]
        mine = off(x, w)[0]
        print(f"  {name}: {mine:.2e} against {once:.2e}, {mine / once:.2f} times, limit {limit}", flush=True)
        assert mine <= limit * once, (name, mine, once)


@pytest.mark.parametrize("scale", [0.37, 0.125])
def test_fp32_scores_far_from_zero(cuda_device, scale):
    """Small whole numbers, so that scores are exact: all near 1600, which scaled is up to 850 in powers of two. A
    row's lse as one float would be off by up to 2^-15 there, and all its weights with it by 2e-5. With
    their difference from it exact to an ulp of itself, weights of 2^-10 and more are off by 10 u at
    most, most by 2 u: 12 u for out and dv, whose roundings average out, 24 u for dq and dk."""
    print(f"[case] fp32, scores near 1600, scale {scale}", flush=True)
    g = torch.Generator().manual_seed(4)
    q, k = (torch.randint(-1, 2, (B, N, heads, D), generator=g).float() for heads in (H, KV))
    q[..., 0] = k[..., 0] = 40.0
    v, dout = (torch.randn(B, N, heads, D, generator=g) for heads in (KV, H))
    q, k, v, dout = (t.to(cuda_device) for t in (q, k, v, dout))
    want = attention64(q, k, v, WINDOW, SINKS, scale, None, dout)
    got = run(q, k, v, dout, window=WINDOW, sinks=SINKS, scale=scale)
    u = UNIT[torch.float32]
    close(got[0], want[0], 12 * u, "out")
    close(got[3], want[3], 12 * u, "dv")
    # the first dim's 40 takes the sum of ds, which is 0 but for roundings, 40 times: left out
    close(got[1][..., 1:], want[1][..., 1:], 24 * u, "dq")
    close(got[2][..., 1:], want[2][..., 1:], 24 * u, "dk")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("scale", [1e-3, 0.11, 0.7])
def test_scales(cuda_device, dtype, scale):
    """Any scale, for rows and for single tokens, with the tolerances of the default one times what larger scores cost."""
    print(f"[case] scale {scale} {dtype}", flush=True)
    i = inputs(cuda_device, "plain", dtype)
    want = attention64(*i[:3], WINDOW, SINKS, scale, None, i[3])
    got = run(*i[:3], i[3], window=WINDOW, sinks=SINKS, scale=scale)
    token = run(i[0][:, -1:], *i[1:3], i[3][:, -1:], window=WINDOW, sinks=SINKS, scale=scale)
    u = UNIT[dtype]
    forward, backward = (64 * u, 128 * u) if dtype == torch.float32 else (4 * u, 8 * u)
    for x, w, name in zip(got, want, ("out", "dq", "dk", "dv")):
        floor = 2.0 ** -25 * w.numel() ** 0.5 / float(w.norm()) if dtype == torch.float16 else 0.0
        close(x, w, (forward if name in ("out", "dv") else backward) + floor, name)
    close(token[0], want[0][:, -1:], forward, "a token")


@pytest.mark.parametrize("shape", [(7, 26, 8, 8, 128), (2, 8, 8, 2, 128), (3, 30, 4, 4, 64)], ids=str)
def test_fp32_weights_near_one_of_few_rows(cuda_device, shape):
    """Few rows go through the kernel for tokens; the backward makes p of its own scores and of that kernel's lse. A
    row's largest weight is near 1 if both round the scores alike, whatever their size (some 100 here): a
    weight is then off by an ulp or two of exp2, its sums of up to 32 terms by as much. 8 u for dv, which is
    most of the first key's; a score rounded otherwise is off by some u of 100 itself."""
    b, n, h, kv, d = shape
    print(f"[case] fp32, weights near 1, {shape}", flush=True)
    g = torch.Generator().manual_seed(5)
    q, k, v, dout = (torch.randn(b, n, heads, d, generator=g) for heads in (h, kv, kv, h))
    s = torch.randn(d, generator=g) * (1.5 * (64 / d) ** 0.5)
    q, k = q + s, k * 0.3
    k[:, :1] += s
    q, k, v, dout = (t.to(cuda_device) for t in (q, k, v, dout))
    want = attention64(q, k, v, None, 0, d ** -0.5, None, dout)
    got = run(q, k, v, dout)
    close(got[3], want[3], 8 * UNIT[torch.float32], "dv")
