"""Routing of logits far below the largest: weights down to fp32's smallest numbers; and of large ones.

u = 2^-24. The differences are exact here (multiples of 1/2 below 128), so a weight is off by the exponential's
3 u, the sum's 36 u and the division's u of itself, 100 u taken, and by two roundings among subnormal
numbers, half of 2^-149 each.
"""

from __future__ import annotations

import pytest
import torch

from mtp_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("T,E,k,dtype", [
    (5, 40, 12, torch.float32), (5, 40, 12, torch.bfloat16), (5, 300, 40, torch.float16), (7, 500, 64, torch.float32),
    (1100, 40, 12, torch.float32), (1100, 200, 16, torch.float16), (1030, 400, 16, torch.bfloat16), (1030, 64, 16, torch.bfloat16)])
def test_weights_among_the_smallest_numbers(T, E, k, dtype, renorm):
    g = torch.Generator().manual_seed(E)
    l = -86.5 - 0.5 * torch.randint(0, 36, (T, E), generator=g)  # -104 .. -86.5
    l[torch.arange(T), torch.randint(0, E, (T,), generator=g)] = 0.0
    l[T // 2] += 20.0
    r = ops.route_tokens(l.to(dtype).cuda(), k, renormalize=renorm)
    x = l.double()
    top, ids = x.sort(dim=1, descending=True, stable=True)
    want = torch.softmax(x, 1).gather(1, ids[:, :k])
    if renorm:
        want = want / want.sum(1, keepdim=True)
    assert torch.equal(r.topk_ids.cpu().long(), ids[:, :k])
    off = (r.topk_weights.cpu().double() - want).abs() / (100 * U * want + 2.0 ** -149)
    worst = float(off.max())
    assert worst <= 1


@pytest.mark.parametrize("T,E,k,dtype", [
    (12, 40, 4, torch.float32), (300, 40, 4, torch.bfloat16), (300, 300, 20, torch.float32),
    (5000, 64, 8, torch.float32), (5000, 64, 8, torch.bfloat16), (70000, 8, 2, torch.float32)])
def test_z_loss_of_large_logits(T, E, k, dtype):
    """Logits of 10^19: their squares' mean is a third of the largest fp32 value, their sum is beyond it. log sum exp
    is the largest logit there (the rest is below its half step), so the loss is off by its own roundings."""
    g = torch.Generator().manual_seed(T)
    l = (1e19 * (1 + 0.02 * torch.rand(T, E, generator=g))).to(dtype)
    r = ops.route_tokens(l.cuda(), k)
    want = l.double().max(1).values.square().mean()
    assert abs(float(r.z_loss) - want) <= 8 * U * want
    assert bool(r.topk_weights.isfinite().all()) and bool(r.balance_loss.isfinite())
