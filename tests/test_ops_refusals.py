"""Refusals of the row sort, the int8 products and the block norm: the wrappers' argument checks and
the entry points' own, none of which launches anything (no GPU needed)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from mtp_amd import _lib, ops
from mtp_amd.weights import Int8Experts

F, I = torch.bfloat16, torch.int32


def z(*shape, dtype=F):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call,error", [
    (lambda: ops.dispatch_tokens(z(4, 8, dtype=torch.float64), z(4, 2, dtype=I), 8), TypeError),
    (lambda: ops.dispatch_tokens(z(4, 8, 1), z(4, 2, dtype=I), 8), ValueError),
    (lambda: ops.dispatch_tokens(z(4, 8), z(4, 2, dtype=torch.int64), 8), TypeError),
    (lambda: ops.dispatch_tokens(z(4, 8), z(3, 2, dtype=I), 8), ValueError),
    (lambda: ops.dispatch_tokens(z(4, 8), z(4, 2, dtype=I), 8), ValueError),  # host tensors
    (lambda: ops.dispatch_tokens(z(4, 8), z(4, 65, dtype=I), 8), ValueError),
    (lambda: ops.dispatch_tokens(z(4, 8), z(4, 2, dtype=I), 0), ValueError),
    (lambda: ops.dispatch_tokens(z(4, 8), z(4, 2, dtype=I), 2 ** 32 + 8), ValueError),
    (lambda: ops.quantize_tokens(z(1, 1).expand(2 ** 32 + 1, 1)), ValueError),
    (lambda: ops.int8_linear(z(4, 16), torch.zeros(1, 16, dtype=torch.int8).expand(2 ** 31, 16),
                             torch.zeros(1).expand(2 ** 31)), ValueError),
    (lambda: ops.combine_tokens(z(8, 8), z(4, 2, dtype=I), z(4, 2)), TypeError),
    (lambda: ops.combine_tokens(z(8, 8), z(4, 2, dtype=I), torch.zeros(4, 3)), ValueError),
    (lambda: ops.combine_tokens(z(7, 8), z(4, 2, dtype=I), torch.zeros(4, 2)), ValueError),
    (lambda: ops.quantize_tokens(z(4, 8, dtype=torch.int32)), TypeError),
    (lambda: ops.quantize_tokens(z(8)), ValueError),
    (lambda: ops.int8_linear(z(4, 32), z(8, 32), torch.zeros(8)), TypeError),
    (lambda: ops.int8_linear(z(4, 32), z(8, 16, dtype=torch.int8), torch.zeros(8)), ValueError),
    (lambda: ops.int8_linear(z(4, 32), z(8, 32, dtype=torch.int8), torch.zeros(7)), ValueError),
    (lambda: ops.int8_linear(z(4, 32), z(8, 32, dtype=torch.int8), torch.zeros(8),
                             bias=torch.zeros(8)), ValueError),
    (lambda: ops.int8_matmul(z(4, 32), torch.zeros(4), z(8, 32, dtype=torch.int8),
                             torch.zeros(8)), TypeError),
    (lambda: ops.int8_matmul(z(4, 32, dtype=torch.int8), torch.zeros(4),
                             z(8, 32, dtype=torch.int8), torch.zeros(8), dtype=torch.int32),
     TypeError),
    (lambda: ops.block_norm(z(4, 8), z(4, 7)), ValueError),
    (lambda: ops.block_norm(z(4, 8), torch.zeros(4, 8)), ValueError),
    (lambda: ops.block_norm(z(4, 8), z(4, 8), post_w=z(7)), ValueError),
    (lambda: ops.block_norm(z(4, 8), z(4, 8), pre_w=torch.zeros(8)), ValueError),
    (lambda: ops.block_norm(z(4, 8), z(4, 8), gate=z(4)), ValueError),
    (lambda: ops.block_norm(z(4, 8), z(4, 8), gate=z(1, 8)), ValueError),
    (lambda: ops.block_norm(z(4, 8), z(4, 8), gate=torch.zeros(8)), ValueError),
])
def test_wrappers_refuse(call, error):
    with pytest.raises(error):
        call()


def _set(E=4, H=64, N=32, dtype=torch.int8):
    q = {"gate": (E, N, H), "up": (E, N, H), "down": (E, H, N)}
    return {k: v for n, s in q.items()
            for k, v in ((n, torch.zeros(s, dtype=dtype)), (n + "_scale", torch.zeros(s[:2])))}


def test_int8_experts_container_refuses():
    Int8Experts(**_set())
    for change in ({"up": torch.zeros(4, 32, 48, dtype=torch.int8)},
                   {"down_scale": torch.zeros(4, 32)},
                   {"gate": torch.zeros(32, 64, dtype=torch.int8)},
                   {"up": torch.zeros(4, 64, 32, dtype=torch.int8).transpose(1, 2)}):
        with pytest.raises(ValueError):
            Int8Experts(**{**_set(), **change})
    with pytest.raises(TypeError):
        Int8Experts(**_set(dtype=torch.uint8))
    with pytest.raises(ValueError, match="multiples of 16"):
        Int8Experts(**_set(H=40))
    with pytest.raises(ValueError, match="512 experts"):
        Int8Experts(**_set(E=513, H=16, N=16))


NULL, SHAPE, UNSUP, WS = (_lib.MOE_ERR_NULL, _lib.MOE_ERR_SHAPE, _lib.MOE_ERR_UNSUPPORTED,
                          _lib.MOE_ERR_WORKSPACE)
A, B, C, D, G, W = (0x1000000 * i for i in range(1, 7))  # never dereferenced


@pytest.mark.parametrize("code,entry,args", [
    (SHAPE, "moe_dispatch_v1", (A, -1, 64, 0, B, 8, 16, None, 0, C, D, G, W)),
    (SHAPE, "moe_dispatch_v1", (A, 4, 64, 0, B, 65, 16, None, 0, C, D, G, W)),
    (SHAPE, "moe_dispatch_v1", (A, 1 << 20, 64, 0, B, 8, 16, None, 0, C, D, G, W)),
    (SHAPE, "moe_dispatch_v1", (A, 4, 64, 0, B, 8, 513, None, 0, C, D, G, W)),
    (SHAPE, "moe_dispatch_v1", (A, 4, 0, 0, B, 8, 16, None, 0, C, D, G, W)),
    (UNSUP, "moe_dispatch_v1", (A, 4, 64, 3, B, 8, 16, None, 0, C, D, G, W)),
    (NULL, "moe_dispatch_v1", (A, 4, 64, 0, B, 8, 16, None, 0, C, D, G, None)),
    (NULL, "moe_dispatch_v1", (None, 0, 64, 0, None, 8, 16, None, 0, None, None, None, None)),
    (WS, "moe_dispatch_v1", (A, 4096, 64, 0, B, 8, 16, None, 0, C, D, G, W)),
    (WS, "moe_dispatch_v1", (A, 4096, 64, 0, B, 8, 16, W + 16, 1 << 30, C, D, G, W)),
    (SHAPE, "moe_dispatch_v1", (A, 4, 64, 0, B, 8, 16, None, 0, A + 64, D, G, W)),
    (NULL, "moe_combine_v1", (A, 4, 8, 64, 0, None, B, C)),
    (SHAPE, "moe_combine_v1", (A, 4, 8, 64, 0, D, B, A + 128)),
    (SHAPE, "moe_combine_v1", (A, 4, 8, 65537, 0, D, B, C)),
    (SHAPE, "moe_combine_v1", (A, 4, 8, 64, 0, C + 64, B, C)),
    (SHAPE, "moe_combine_v1", (A, 4, 8, 64, 0, D, C + 64, C)),
    (SHAPE, "moe_dispatch_v1", (A, 4, 64, 0, B, 8, 16, None, 0, C, D, G, B)),
    (SHAPE, "moe_dispatch_v1", (A, 4, 64, 0, B, 8, 16, None, 0, C, B + 64, G, W)),
    (SHAPE, "moe_dispatch_v1", (A, 600, 64, 0, B, 8, 16, A + 1024, 1 << 30, C, D, G, W)),
    (UNSUP, "moe_combine_v1", (A, 4, 8, 64, -1, D, B, C)),
    (NULL, "moe_combine_backward_v1", (A, B, 4, 8, 64, 0, C, D, None, None)),
    (NULL, "moe_combine_backward_v1", (A, None, 4, 8, 64, 0, C, D, None, G)),
    (NULL, "moe_combine_backward_v1", (A, B, 4, 8, 64, 0, C, None, G, None)),
    (SHAPE, "moe_combine_backward_v1", (A, B, 4, 8, 64, 0, C, D, B, None)),
    (SHAPE, "moe_combine_backward_v1", (A, B, 4, 8, 64, 0, C, D, G, D)),
    (SHAPE, "moe_combine_backward_v1", (A, B, 4, 8, 64, 0, C, D, G, C)),
    (SHAPE, "moe_combine_backward_v1", (A, B, 4, 8, 64, 0, C, D, G, G + 256)),
    (SHAPE, "moe_quantize_tokens_v1", (A, 4, 65537, 0, B, C)),
    (SHAPE, "moe_quantize_tokens_v1", (A, 4, 64, 0, A + 8, C)),
    (SHAPE, "moe_quantize_tokens_v1", (A, 4, 64, 0, B, B + 128)),
    (SHAPE, "moe_quantize_tokens_v1", (A, 1 << 22, 16384, 0, B, C)),
    (NULL, "moe_quantize_tokens_v1", (A, 4, 64, 0, None, C)),
    (SHAPE, "moe_int8_matmul_v1", (A, B, 4, 40, C, D, 8, None, 0, G)),
    (SHAPE, "moe_int8_matmul_v1", (A, B, 4, 65552, C, D, 8, None, 0, G)),
    (SHAPE, "moe_int8_matmul_v1", (A, B, 1 << 20, 2048, C, D, 8, None, 0, G)),
    (SHAPE, "moe_int8_matmul_v1", (A, B, 4, 2048, C, D, 1 << 20, None, 0, G)),
    (SHAPE, "moe_int8_matmul_v1", (A, B, 4, 64, C + 8, D, 8, None, 0, G)),
    (SHAPE, "moe_int8_matmul_v1", (A, B, 4, 64, C, D, 8, None, 0, A)),
    (NULL, "moe_int8_matmul_v1", (A, None, 4, 64, C, D, 8, None, 0, G)),
    (UNSUP, "moe_int8_matmul_v1", (A, B, 4, 64, C, D, 8, None, 7, G)),
    (WS, "moe_int8_linear_v1", (A, 40, 64, 0, B, C, 8, None, D, 16, G)),
    (WS, "moe_int8_linear_v1", (A, 40, 64, 0, B, C, 8, None, None, 1 << 20, G)),
    (WS, "moe_int8_linear_v1", (A, 40, 64, 0, B, C, 8, None, D + 16, 1 << 20, G)),
    (SHAPE, "moe_int8_linear_v1", (A, 4, 64, 0, B, C, 8, None, D, 1 << 20, A)),
    (SHAPE, "moe_block_norm_v1", (A, B, 4, 8193, 0, None, None, 0, 1.0, 1.0, None, 1e-6, C, None)),
    (SHAPE, "moe_block_norm_v1", (A, B, 4, 64, 0, None, None, 0, 1.0, 1.0, None, -1.0, C, None)),
    (SHAPE, "moe_block_norm_v1", (A, B, 4, 64, 0, None, None, 0, 1.0, 1.0, None, 1e-6, A, None)),
    (SHAPE, "moe_block_norm_v1", (A, B, 4, 64, 0, None, None, 0, 1.0, 1.0, D, 1e-6, C, C)),
    (NULL, "moe_block_norm_v1", (A, B, 4, 64, 0, None, None, 2, 1.0, 1.0, None, 1e-6, C, None)),
    (NULL, "moe_block_norm_v1", (A, B, 4, 64, 0, None, None, 0, 1.0, 1.0, D, 1e-6, C, None)),
    (UNSUP, "moe_block_norm_v1", (A, B, 4, 64, 0, None, D, 4, 1.0, 1.0, None, 1e-6, C, None)),
    (WS, "moe_block_norm_backward_v1", (A, B, 4, 64, 0, C, None, 0, 1.0, 1.0, None, 1e-6, D, None,
                                        None, 0, None, None, G, None, None)),
    (NULL, "moe_block_norm_backward_v1", (A, B, 4, 64, 0, None, None, 0, 1.0, 1.0, None, 1e-6, D,
                                          None, W, 1 << 20, None, None, G, None, None)),
    (SHAPE, "moe_block_norm_backward_v1", (A, B, 4, 64, 0, None, None, 0, 1.0, 1.0, None, 1e-6, D,
                                           None, None, 0, A, None, None, None, None)),
])
def test_entry_points_refuse(code, entry, args):
    lib = _lib.load()
    assert getattr(lib, entry)(*args, None) == code, lib.moe_w4a16_last_error()


@pytest.mark.parametrize("change,code", [
    ({"gate": None}, NULL), ({"num_experts": 513}, SHAPE), ({"hidden": 40}, SHAPE),
    ({"intermediate": 24}, SHAPE), ({"up": B + 8}, SHAPE)])
def test_int8_experts_entry_refuses(change, code):
    lib = _lib.load()
    fields = {"gate": A, "up": B, "down": C, "gate_scale": A, "up_scale": B, "down_scale": C,
              "num_experts": 8, "hidden": 64, "intermediate": 32}
    good = _lib.Int8Set(**fields)
    need = lib.moe_int8_experts_workspace_bytes_v1(4, 2, ctypes.byref(good), 0)
    assert need > 0
    assert lib.moe_int8_experts_v1(D, 4, 0, G, W, 2, ctypes.byref(good), 0x10000000, need - 1, D,
                                   None) == WS
    assert lib.moe_int8_experts_v1(D, 4, 0, G, W, 2, ctypes.byref(good), D, need, G, None) == SHAPE
    assert lib.moe_int8_experts_v1(D, 4, 0, G, W, 65, ctypes.byref(good), 0x10000000, 1 << 30, D,
                                   None) == SHAPE
    bad = _lib.Int8Set(**{**fields, **change})
    assert lib.moe_int8_experts_workspace_bytes_v1(4, 2, ctypes.byref(bad), 0) == -1
    assert lib.moe_int8_experts_v1(D, 4, 0, G, W, 2, ctypes.byref(bad), 0x10000000, 1 << 30, D,
                                   None) == code


def test_workspace_queries_refuse_sizes():
    lib = _lib.load()
    assert lib.moe_dispatch_workspace_bytes_v1(-1, 8, 16) == -1
    assert lib.moe_dispatch_workspace_bytes_v1(8, 8, 16) == 0
    assert lib.moe_int8_linear_workspace_bytes_v1(-1, 64) == -1
    assert lib.moe_int8_linear_workspace_bytes_v1(4, 64) == 0
    assert lib.moe_int8_linear_workspace_bytes_v1(40, 64) > 0
    assert lib.moe_block_norm_workspace_bytes_v1(4, 8193) == -1
