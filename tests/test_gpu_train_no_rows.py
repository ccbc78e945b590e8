"""The losses of tuning over no rows (a batch that was filtered to nothing), with gradients as without."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from tests.test_block_abi import refused
from tests.test_train_abi import Policy, _lib, changed, logits  # noqa: F401  (a fixture)


def test_statistics_of_no_rows_may_be_null(lib):
    """A tensor without elements has no address, one count has: the call gets past that check (CPU only: the next one,
    of the workspace, ends it)."""
    fake = ctypes.c_void_p(4096)
    for reduction in (0, 1):
        for stats, slope in ((None, None), (fake, None), (None, fake), (fake, fake)):
            p = changed(Policy(logits(0), 4096, 4096, 4096, 0.8, 1.2, 0.1), {})
            refused(lib, lib.isa_train_policy_forward(p, reduction, fake, None, stats, slope, fake, fake, 16, None),
                    "workspace too small")


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0,), (0, 3), (3, 0)], ids=str)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_policy_of_no_rows(cuda_device, shape, reduction):
    from isa.kernels.transformer_block import policy_loss

    t = torch.zeros(shape, dtype=torch.int64, device=cuda_device)
    f = torch.zeros(shape, device=cuda_device)
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.zeros(*shape, 50, dtype=dtype, device=cuda_device)
        leaf = x.clone().requires_grad_(True)
        print(f"[case] policy {shape} {reduction} {dtype}", flush=True)
        loss, logp = policy_loss(leaf, t, f, f, ref_logp=f, kl=0.1, reduction=reduction)
        (dx,) = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
        assert logp.shape == shape and dx.shape == x.shape and dx.dtype == dtype
        assert loss.shape == (shape if reduction == "none" else ())
        plain = policy_loss(x, t, f, f, ref_logp=f, kl=0.1, reduction=reduction)[0]
        assert torch.equal(torch.nan_to_num(loss.detach(), 5.0), torch.nan_to_num(plain, 5.0))
        if reduction != "none":
            assert math.isnan(float(loss)) if reduction == "mean" else float(loss) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 3), (4, 0)], ids=str)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_preference_of_no_rows(cuda_device, shape, reduction):
    from isa.kernels.transformer_block import preference_loss

    t = torch.zeros(shape, dtype=torch.int64, device=cuda_device)
    leaf = torch.zeros(*shape, 50, device=cuda_device, requires_grad=True)
    print(f"[case] preference {shape} {reduction}", flush=True)
    loss, _ = preference_loss(leaf, t, torch.zeros(shape[0], device=cuda_device), reduction=reduction)
    (dx,) = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    assert dx.shape == leaf.shape
    if shape[0]:  # margins of 0 in two pairs
        want = math.log(2.0) * (2.0 if reduction == "sum" else 1.0)
        assert float((loss - want).abs().max()) <= 1e-6
