"""What the C entry points of the row sort, the int8 products and the block norm check before a launch:
pointers that a kernel would read whatever the sizes, memory that two arguments share, and sizes past
a launch. Nothing here launches anything (no GPU needed)."""

from __future__ import annotations

import pytest

from mtp_amd import _lib

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
