"""Refusals of the routing's arguments that need no GPU."""

from __future__ import annotations

import pytest
import torch

from mtp_amd import ops


@pytest.mark.parametrize("top_k", [2.5, 1.999, 7.0000001, float("nan"), float("inf")])
def test_a_fractional_top_k_is_refused(top_k):
    with pytest.raises(ValueError, match="top_k"):
        ops.route_tokens(torch.zeros(4, 8), top_k)


@pytest.mark.parametrize("top_k", [2, 2.0, True])
def test_a_whole_top_k_gets_as_far_as_the_device(top_k):
    with pytest.raises(ValueError, match="device tensors"):
        ops.route_tokens(torch.zeros(4, 8), top_k)
