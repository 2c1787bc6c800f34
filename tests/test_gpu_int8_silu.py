"""The int8 experts' SiLU in fp32."""

from __future__ import annotations

import pytest
import torch

from mtp_amd import ops
from mtp_amd.weights import Int8Experts

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def test_silu_in_fp32():
    """fp32 experts keep fp32's precision in h = silu(g) u. Each expert has one channel whose up
    projection is not zero, so that its h is the row's largest value a, 127 as an integer, and the
    output 127 (a / 127): 2 half steps off a. h itself: e^-g 1 ulp (2), the sum, the quotient and the
    product one each: 7 in all."""
    E, H, I = 320, 16, 16
    gate, up, down = (torch.zeros(E, n, 16, dtype=torch.int8) for n in (I, I, H))
    gate[:, 0, 0], up[:, 0, 0], down[:, :, 0] = 127, 1, 1
    gs = torch.linspace(-80.0, 80.0, E) / 16129.0
    ex = Int8Experts(gate, gs[:, None].repeat(1, I), up, torch.full((E, I), 1.0 / 128), down,
                     torch.ones(E, H))
    x = torch.zeros(E, H)
    x[:, 0] = 127.0  # quantised to 127 with a scale of 1
    ids = torch.arange(E, dtype=torch.int32)[:, None]
    got = ops.int8_experts(x.cuda(), ids.cuda(), torch.ones(E, 1).cuda(), ex.to("cuda")).cpu().double()
    g = (torch.tensor(16129.0) * gs).double()
    want = (g * torch.sigmoid(g) * (127.0 / 128))[:, None]
    err = (got - want).abs() / want.abs()
    assert float(err.max()) <= 7.01 * U, float(err.max()) / U
