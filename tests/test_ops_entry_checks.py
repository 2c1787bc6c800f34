"""What the C entry points of the row sort, the int8 products and the block norm check before a launch:
pointers that a kernel would read whatever the sizes, memory that two arguments share, and sizes past
a launch. Nothing here launches anything (no GPU needed)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from mtp_amd import _lib, ops
from mtp_amd.weights import Int8Experts

NULL, SHAPE = _lib.MOE_ERR_NULL, _lib.MOE_ERR_SHAPE
A, B, C, D, G, P, W = (0x1000000 * i for i in range(1, 8))  # never dereferenced


def code_of(entry, *args):
    return getattr(_lib.load(), entry)(*args, None)


def norm_backward(T, H, *, post=None, gate=None, kind=0, pre=None, dr=P, dx=None, ws=W, dy=None,
                  dres=None, dpost=None, dgate=None, dpre=None, y=A, r=B, dtype=0):
    return code_of("moe_block_norm_backward_v1", y, r, T, H, dtype, post, gate, kind, 1.0, 1.0, pre,
                   1e-6, dr, dx, ws, 1 << 22, dy, dres, dpost, dgate, dpre)


@pytest.mark.parametrize("grads", [{"dgate": D}, {"dpost": D, "post": C}, {"dpre": D, "pre": C, "dx": G}])
def test_block_norm_backward_refuses_a_missing_channel_gate_without_tokens(grads):
    """The weights' gradients are written (zeros) also where there are no tokens, and the kernel that
    does it reads a channel gate, [hidden], ahead of its first row."""
    assert norm_backward(0, 64, kind=2, gate=None, **grads) == NULL


@pytest.mark.parametrize("shared", ["q_scale", "w_scale", "bias"])
def test_int8_matmul_refuses_out_over_scales_and_bias(shared):
    """Every workgroup loads the scales and the bias for itself: one could read another's results."""
    at = {"q_scale": B, "w_scale": D, "bias": P, "out": G}
    at[shared] = G + 16
    assert code_of("moe_int8_matmul_v1", A, at["q_scale"], 40, 64, C, at["w_scale"], 32, at["bias"], 0,
                   G) == SHAPE


@pytest.mark.parametrize("T", [2, 40])  # with and without a workspace
@pytest.mark.parametrize("shared", ["w_scale", "bias"])
def test_int8_linear_refuses_out_over_scales_and_bias(T, shared):
    at = {"w_scale": D, "bias": P}
    at[shared] = G + 16
    assert code_of("moe_int8_linear_v1", A, T, 64, 0, C, at["w_scale"], 32, at["bias"], W, 1 << 20,
                   G) == SHAPE


@pytest.mark.parametrize("shared", ["w", "w_scale", "bias"])
def test_int8_linear_refuses_a_workspace_over_the_weights(shared):
    """The quantised rows would be written over what the product reads."""
    at = {"w": C, "w_scale": D, "bias": P}
    at[shared] = W + 256
    assert code_of("moe_int8_linear_v1", A, 40, 64, 0, at["w"], at["w_scale"], 32, at["bias"], W, 1 << 20,
                   G) == SHAPE


@pytest.mark.parametrize("shared", ["gate", "up", "down", "gate_scale", "up_scale", "down_scale"])
def test_int8_experts_refuse_a_workspace_over_the_weights(shared):
    """The workspace's rows would be written over what the products read."""
    big = 0x10000000
    ptrs = {n: big + 0x1000000 * i for i, n in enumerate(
        ("gate", "up", "down", "gate_scale", "up_scale", "down_scale"))}
    ptrs[shared] = W + 256
    ex = _lib.Int8Set(**ptrs, num_experts=8, hidden=64, intermediate=32)
    assert code_of("moe_int8_experts_v1", A, 4, 0, B, C, 2, ctypes.byref(ex), W, 1 << 20, D) == SHAPE


def norm(T, H, *, post=None, gate=None, kind=0, pre=None, r=C, x=None):
    return code_of("moe_block_norm_v1", A, B, T, H, 0, post, gate, kind, 1.0, 1.0, pre, 1e-6, r, x)


@pytest.mark.parametrize("over", [C, D])  # the residual stream, the next block's input
def test_block_norm_refuses_outputs_over_weights_and_gates(over):
    """Weights and gates are read again for each row, while other rows are written."""
    at = over + 8 * 64 * 2 - 2  # the outputs' last element
    assert norm(8, 64, post=at, pre=P, x=D) == SHAPE
    assert norm(8, 64, post=P, pre=at, x=D) == SHAPE
    assert norm(8, 64, pre=P, x=D, gate=at, kind=1) == SHAPE
    assert norm(8, 64, pre=P, x=D, gate=at, kind=2) == SHAPE
    assert norm(8, 64, pre=P, x=D, gate=at, kind=3) == SHAPE


BACKWARD = {  # a valid call of 8 x 64 bf16 with every input and output
    "y": A, "r": B, "post": C, "gate": D, "pre": G, "dr": P, "dx": W, "ws": 0x20000000,
    "dy": 0x11000000, "dres": 0x12000000, "dpost": 0x13000000, "dgate": 0x14000000, "dpre": 0x15000000}


@pytest.mark.parametrize("kind", [1, 2, 3])
@pytest.mark.parametrize("out", ["dy", "dres", "dpost", "dgate", "dpre", "ws"])
def test_block_norm_backward_refuses_shared_memory(out, kind):
    """A gradient, or the workspace's partial sums, over an input or over each other: rows, weights and
    partial sums are read while others are written."""
    for other in BACKWARD:
        if other != out:
            # the output's first byte is the other's; the workspace begins on 256 bytes
            call = {**BACKWARD, **({other: BACKWARD[out]} if out == "ws" else {out: BACKWARD[other]})}
            assert norm_backward(8, 64, kind=kind, **call) == SHAPE, other


def test_block_norm_backward_refuses_partly_shared_memory():
    last = 8 * 64 * 2 - 2  # a gradient's last element
    for out, other in (("dy", "pre"), ("dres", "gate"), ("dgate", "post"), ("dy", "dpost")):
        call = {**BACKWARD, other: BACKWARD[out] + last}
        assert norm_backward(8, 64, kind=3, **call) == SHAPE, (out, other)
    need = _lib.load().moe_block_norm_workspace_bytes_v1(8, 64)
    assert norm_backward(8, 64, kind=2, **{**BACKWARD, "dr": BACKWARD["ws"] + need - 4}) == SHAPE


@pytest.mark.parametrize("T", [4, 4096])  # without and with a workspace
def test_dispatch_refuses_outputs_over_each_other(T):
    """Workgroups write rows while others still read the tables and the workspace's counts."""
    outs = {"rows": 0x40000000, "offsets": 0x51000000, "row_slot": 0x52000000, "slot_row": 0x53000000}
    if T > 512:
        outs["ws"] = 0x54000000
    for out in outs:
        for other in outs:
            if other != out:
                o = {**outs, out: outs[other] + (0 if out == "ws" else 4)}
                assert code_of("moe_dispatch_v1", A, T, 64, 0, B, 8, 16, o.get("ws"), 1 << 20, o["rows"],
                               o["offsets"], o["row_slot"], o["slot_row"]) == SHAPE, (out, other)


@pytest.mark.parametrize("hidden", [8, 512, 513, 4097])
def test_block_norm_workspace_of_the_most_tokens(hidden):
    """Many tokens share a fixed number of workgroups: from there on the size stays."""
    query = _lib.load().moe_block_norm_workspace_bytes_v1
    assert query(2 ** 31 - 1, hidden) == query(1 << 20, hidden) > query(1, hidden)


def test_int8_linear_refuses_more_rows_than_a_launch():
    """Quantising takes 64 threads a row, of which a launch has fewer than 2^32: rows of 16 columns
    pass that below the operands' 2 GiB."""
    big = 1 << 40
    assert code_of("moe_int8_linear_v1", A, 1 << 26, 16, 0, big, big + 4096, 16, None, 2 * big, 1 << 40,
                   3 * big) == SHAPE


@pytest.mark.parametrize("T,k", [(2 ** 32 + 8, 2), (8, 2 ** 32 + 2), (2 ** 31, 1), (-1, 2), (8, 0)])
def test_int8_experts_workspace_query_refuses_sizes(T, k):
    """Sizes are int32 in the library, and passing a larger one cuts it off."""
    ex = Int8Experts(*(t for n, K in ((32, 64), (32, 64), (64, 32)) for t in (
        torch.zeros(4, n, K, dtype=torch.int8), torch.ones(4, n))))
    assert ops.int8_experts_workspace_bytes(8, 2, ex) > 0
    with pytest.raises(ValueError):
        ops.int8_experts_workspace_bytes(T, k, ex)
