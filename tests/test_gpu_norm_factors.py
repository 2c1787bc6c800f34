"""block_norm's factors where the order and width of their sums decide, and the weights' gradients of
no tokens."""

from __future__ import annotations

import pytest
import torch

from mtp_amd import _lib, ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def spiked(H):
    """A row of one 1 and, in every other group of 8 columns, one 2^-15: squares 1 and 2^-30. A thread's
    own sum (of 8 columns) is exact; an fp32 sum over the threads that starts at the 1 loses all others,
    2^-30 (H / 8 - 1) of the sum and half as much of the factor: 2^-22 for 4096 columns."""
    row = torch.zeros(2, H)
    row[:, 8::8] = 2.0 ** -15
    row[:, 0] = 1.0
    return row, (1 + (H // 8 - 1) * 2.0 ** -30) / H


@pytest.mark.parametrize("H", [4096, 8192])
def test_squares_are_summed_in_64_bits(H):
    """Each value below is a norm's factor times powers of two, so it is off by the factor's rounding
    alone, half a step; in fp32 sums by 4 and 8 of them more."""
    row, mean = spiked(H)
    want = mean ** -0.5
    zero, w = torch.zeros_like(row).cuda(), torch.zeros(H).cuda()

    def check(value):
        assert bool(((value.double() - want).abs() <= (1 + 2.0 ** -10) * U * want).all())

    r, x = ops.block_norm(zero, row.cuda(), pre_w=w, eps=0.0)
    check(x[:, 0])
    r, _ = ops.block_norm(row.cuda(), zero, post_w=w, eps=0.0)
    check(r[:, 0])
    # gradients that enter at column 1, where the row is 0, have no mean to subtract
    unit = torch.zeros_like(row).cuda()
    unit[:, 1] = 1.0
    leaf = row.cuda().requires_grad_()
    _, x = ops.block_norm(zero, leaf, pre_w=w, eps=0.0)
    check(torch.autograd.grad(x, leaf, unit)[0][:, 1])
    r, _ = ops.block_norm(leaf, zero, post_w=w, eps=0.0)
    check(torch.autograd.grad(r, leaf, unit)[0][:, 1])


@pytest.mark.parametrize("H", [40, 2048, 8191])
def test_weight_gradients_of_no_tokens(H):
    """The entry point writes zeros for the weights and a channel gate, its only outputs then."""
    lib = _lib.load()
    w = torch.ones(H, device="cuda")
    need = lib.moe_block_norm_workspace_bytes_v1(0, H)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    grads = [torch.full((H,), float("nan"), device="cuda") for _ in range(3)]
    e = torch.empty(64, device="cuda")  # no row of it is read
    code = lib.moe_block_norm_backward_v1(
        None, e.data_ptr(), 0, H, 2, w.data_ptr(), w.data_ptr(), 2, 1.0, 1.0, w.data_ptr(), 1e-6, None,
        e.data_ptr(), ws.data_ptr(), need, None, None, *(g.data_ptr() for g in grads),
        torch.cuda.current_stream().cuda_stream)
    assert code == 0, lib.moe_w4a16_last_error()
    assert all(float(g.abs().sum()) == 0.0 for g in grads)
